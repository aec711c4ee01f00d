// 8-bit activation checkpoints: equss_ckpt_pack writes an activation as codes and scale bytes (ckpt.h), equss_ckpt_unpack reads
// it back.  Both are one pass over memory and bound by it: a lane owns 16 bytes of the activation (4 channels in fp32, 8 in 16
// bits), so that a wave reads and writes whole kilobytes; 8 or 4 lanes share a block of 32, whose largest magnitude is 3 or 2
// lane exchanges.
//
// Per block: k is the smallest integer >= -110 for which the largest magnitude, times 2^-k and rounded, does not pass 127
// (int8) or 448 (e4m3).  With e = floor(log2(amax)), amax 2^-(e-6) lies in [64, 128) and amax 2^-(e-8) in [256, 512): the
// exponent is right as it is unless the mantissa rounds past the end (127.5 up; above 464, the middle between 448 and the 480
// that e4m3 does not have), where it is one more.  Every code is then off by half a step at most; none saturates.
// At the top of fp32 and bf16 the raised exponent makes the largest codes 64 or 256 times 2^k = 2^128: an infinity, as rounding
// to fewer bits has it anywhere (a cap would keep such a value finite at the cost of a whole step).
#include "ckpt.h"

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4u2 __attribute__((ext_vector_type(4), aligned(2)));

constexpr int kThreads = 256;

template <int T> struct Elem;    // 0 fp32, 1 bf16, 2 fp16
template <> struct Elem<0> { typedef float type; };
template <> struct Elem<1> { typedef u16 type; };
template <> struct Elem<2> { typedef _Float16 type; };

template <int T>
__device__ __forceinline__ float to_f32(typename Elem<T>::type v) {
    if constexpr (T == 0) return v;
    else if constexpr (T == 1) return equss::bf2f(v);
    else return (float)v;
}

template <int T> constexpr int kVec = T == 0 ? 4 : 8;      // channels a lane

// a lane's channels of a row; the rows of an odd width start at any element, which global loads take as they are
template <int T>
__device__ __forceinline__ void load_vec(const typename Elem<T>::type* p, float (&x)[kVec<T>]) {
    if constexpr (T == 0) {
        const f32x4u a = *reinterpret_cast<const f32x4u*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i];
    } else {
        const u32x4u2 w = *reinterpret_cast<const u32x4u2*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == 1) {
                x[2 * i] = equss::bits_as<float>(w[i] << 16);
                x[2 * i + 1] = equss::bits_as<float>(w[i] & 0xffff0000u);
            } else {
                typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
                const f16x2_t h = equss::bits_as<f16x2_t>(w[i]);
                x[2 * i] = (float)h.x;
                x[2 * i + 1] = (float)h.y;
            }
        }
    }
}

template <int T>
__device__ __forceinline__ void store_vec(typename Elem<T>::type* p, const float (&x)[kVec<T>]) {
    if constexpr (T == 0) {
        f32x4u a;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = x[i];
        *reinterpret_cast<f32x4u*>(p) = a;
    } else {
        u32x4u2 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == 1) w[i] = equss::pack_bf16(x[2 * i], x[2 * i + 1]);
            else {
                typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
                w[i] = __builtin_bit_cast(uint32_t, f16x2_t{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
            }
        }
        *reinterpret_cast<u32x4u2*>(p) = w;
    }
}

// A workgroup walks rows_wg rows in units of a lane's channels, units_row of them a row (padded to whole blocks).  A unit's row within the
// workgroup's rows is unit / units_row by one high multiplication: magic = ceil(2^32 / units_row) is exact while
// unit * units_row < 2^32; rows of more units than that have a workgroup to themselves (magic = 0).
struct Walk {
    int64_t rows;
    int width, units_row, rows_wg;
    uint32_t magic;
};

__device__ __forceinline__ void place(const Walk& w, int vec, int64_t row0, uint32_t unit, int64_t& row, int& col) {
    const uint32_t r = __umulhi(unit, w.magic);
    row = row0 + r;
    col = (int)(unit - r * (uint32_t)w.units_row) * vec;
}

template <int T, bool E4M3, bool KEEP>
__global__ __launch_bounds__(kThreads) void ckpt_pack_kernel(const typename Elem<T>::type* __restrict__ x, int64_t ld_x,
                                                            uint8_t* __restrict__ codes, int64_t ld_codes,
                                                            uint8_t* __restrict__ scales, int64_t ld_scales, const Walk w) {
    constexpr int V = kVec<T>, LANES = equss::kCkptBlock / V;
    const int64_t row0 = (int64_t)blockIdx.x * w.rows_wg;
    const int64_t left = w.rows - row0;
    const uint32_t units = (uint32_t)((left < w.rows_wg ? left : w.rows_wg) * w.units_row);
    // units_row is a multiple of a block's LANES and a workgroup starts with a row: these lanes are neighbours, all in or all out
    for (uint32_t u = threadIdx.x; u < units; u += kThreads) {
        int64_t row;
        int col;
        place(w, V, row0, u, row, col);
        const typename Elem<T>::type* src = x + row * ld_x + col;
        float v[V];
        if (col + V <= w.width) load_vec<T>(src, v);
        else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = col + i < w.width ? to_f32<T>(src[i]) : 0.f;
        }
        // the largest magnitude as an integer: the bits of non-negative floats order like their values, infinity and NaN on top
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const uint32_t a = __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu;
            m = a > m ? a : m;
        }
#pragma unroll
        for (int o = 1; o < LANES; o *= 2) {
            const uint32_t other = (uint32_t)__shfl_xor((int)m, o, 64);
            m = other > m ? other : m;
        }
        const bool lost = m >= 0x7f800000u;
        int k = (int)(m >> 23) - 127 - (E4M3 ? 8 : 6);
        k = k < equss::kCkptMinExp ? equss::kCkptMinExp : k;
        const float peak = __builtin_bit_cast(float, m) * equss::ckpt_scale((uint32_t)(127 - k));
        if (E4M3 ? peak > 464.f : peak >= 127.5f) ++k;
        const float inv = equss::ckpt_scale((uint32_t)(127 - k));
        uint32_t out[V / 4];
#pragma unroll
        for (int h = 0; h < V / 4; ++h) {
            float s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = v[4 * h + i] * inv;
            if constexpr (E4M3) {
                float c[4];
                // (448..464 rounds to 448; the conversion's own rounding there would be to a code that e4m3 does not have)
#pragma unroll
                for (int i = 0; i < 4; ++i) c[i] = fminf(fmaxf(s[i], -448.f), 448.f);
                int p = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
                p = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], p, true);
                out[h] = (uint32_t)p;
                if constexpr (KEEP) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (v[4 * h + i] != 0.f && ((out[h] >> (8 * i)) & 0x7fu) == 0) out[h] |= 1u << (8 * i);
                }
            } else {
                out[h] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    int q = (int)rintf(s[i]);
                    if constexpr (KEEP) {
                        if (q == 0 && v[4 * h + i] != 0.f) q = v[4 * h + i] < 0.f ? -1 : 1;   // (v: a subnormal's s may be 0)
                    }
                    out[h] |= ((uint32_t)q & 0xffu) << (8 * i);
                }
            }
        }
        if (lost) {
#pragma unroll
            for (int h = 0; h < V / 4; ++h) {
                out[h] = 0;
                if constexpr (KEEP) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        out[h] |= (v[4 * h + i] > 0.f ? (E4M3 ? 0x7fu : 1u) : v[4 * h + i] < 0.f ? 0xffu : 0u) << (8 * i);
                }
            }
        }
        uint8_t* dst = codes + row * ld_codes + col;
        if constexpr (V == 4) *reinterpret_cast<uint32_t*>(dst) = out[0];
        else *reinterpret_cast<uint2*>(dst) = make_uint2(out[0], out[V / 4 - 1]);
        if ((u & (LANES - 1)) == 0) scales[row * ld_scales + col / equss::kCkptBlock] = (uint8_t)(lost ? equss::kCkptNanByte : k + 127);
    }
}

template <int T, bool E4M3>
__global__ __launch_bounds__(kThreads) void ckpt_unpack_kernel(const uint8_t* __restrict__ codes, int64_t ld_codes,
                                                              const uint8_t* __restrict__ scales, int64_t ld_scales,
                                                              typename Elem<T>::type* __restrict__ out, int64_t ld_out, const Walk w) {
    constexpr int V = kVec<T>;
    const int64_t row0 = (int64_t)blockIdx.x * w.rows_wg;
    const int64_t left = w.rows - row0;
    const uint32_t units = (uint32_t)((left < w.rows_wg ? left : w.rows_wg) * w.units_row);
    for (uint32_t u = threadIdx.x; u < units; u += kThreads) {
        int64_t row;
        int col;
        place(w, V, row0, u, row, col);
        if (col >= w.width) continue;
        const uint32_t* q = reinterpret_cast<const uint32_t*>(codes + row * ld_codes + col);
        uint32_t c[V / 4];
        if constexpr (V == 4) c[0] = *q;
        else {
            const uint2 w2 = *reinterpret_cast<const uint2*>(q);
            c[0] = w2.x;
            c[V / 4 - 1] = w2.y;
        }
        const float s = equss::ckpt_value_scale(scales[row * ld_scales + col / equss::kCkptBlock]);
        float v[V];
#pragma unroll
        for (int h = 0; h < V / 4; ++h) {
            const f32x4 d = equss::ckpt_decode4<E4M3>(c[h]);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * h + i] = d[i] * s;
        }
        typename Elem<T>::type* dst = out + row * ld_out + col;
        if (col + V <= w.width) store_vec<T>(dst, v);
        else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (col + i < w.width) {
                    if constexpr (T == 0) dst[i] = v[i];
                    else if constexpr (T == 1) dst[i] = equss::f2bf(v[i]);
                    else dst[i] = (_Float16)v[i];
                }
        }
    }
}

int checks(const char* what, const void* x, int type, int64_t ld, const void* codes, int64_t ld_codes, const void* scales,
           int64_t ld_scales, int64_t rows, int width, int fmt) {
    if (rows < 0 || width <= 0) return equss::fail(EQUSS_E_SHAPE, "%s: rows=%lld width=%d", what, (long long)rows, width);
    if (type < EQUSS_F32 || type > EQUSS_F16 || (fmt != EQUSS_CKPT_INT8 && fmt != EQUSS_CKPT_E4M3))
        return equss::fail(EQUSS_E_UNSUPPORTED, "%s: element type %d, format %d", what, type, fmt);
    if (width > (1 << 19)) return equss::fail(EQUSS_E_UNSUPPORTED, "%s: width %d (at most 524288)", what, width);
    if (rows == 0) return EQUSS_OK;
    if (!x || !codes || !scales) return equss::fail(EQUSS_E_NULL, "%s: null pointer argument", what);
    const int64_t padded = ((int64_t)width + equss::kCkptBlock - 1) / equss::kCkptBlock * equss::kCkptBlock;
    if (ld < width || ld_codes < padded || (ld_codes % equss::kCkptBlock) != 0 || ((uintptr_t)codes % 16) != 0 ||
        ld_scales < padded / equss::kCkptBlock || ((uintptr_t)x % (type == EQUSS_F32 ? 4 : 2)) != 0)
        return equss::fail(EQUSS_E_ALIGN, "%s: codes 16-byte aligned with a leading dimension that is a multiple of 32 and holds %lld, "
                           "scales %lld to a row, rows of %d elements", what, (long long)padded, (long long)(padded / equss::kCkptBlock), width);
    return EQUSS_OK;
}

// Four units a lane (102400 x 768 bf16, int8: 44 us; 45 with two, 46 with eight, 53 with sixteen), and > 256 workgroups from a
// megabyte on.  Measured at 102400 rows: 768 bf16 written in 43 us (5.5 TB/s of its 238 MB) and read back in 38 us (6.3 TB/s),
// 1024 fp32 in 96 and 92 us (5.5 and 5.8 TB/s of 531 MB; 104 and 142 us with eight channels a lane there too, whose two loads
// and stores leave every other 16 bytes to the next instruction); a copy of 1 GiB runs at 5.15 TB/s.
bool walk(Walk& w, int64_t rows, int width, int type, int64_t& grid) {
    const int vec = type == EQUSS_F32 ? 4 : 8;
    w.rows = rows;
    w.width = width;
    w.units_row = (width + equss::kCkptBlock - 1) / equss::kCkptBlock * (equss::kCkptBlock / vec);
    int64_t r = 4 * kThreads / w.units_row;
    const int64_t spread = (rows + 1023) / 1024;   // few rows: as many workgroups as rows
    if (r > spread) r = spread;
    if (r < 1) r = 1;
    while ((rows + r - 1) / r > equss::max_blocks(kThreads)) r *= 2;
    w.rows_wg = (int)r;
    w.magic = r == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + w.units_row - 1) / w.units_row);
    grid = (rows + r - 1) / r;
    return (uint64_t)r * w.units_row * w.units_row < ((uint64_t)1 << 32) || r == 1;
}

}  // namespace

extern "C" int equss_ckpt_pack(const void* x, int type, int64_t ld_x, void* codes, int64_t ld_codes, void* scales, int64_t ld_scales,
                               int64_t rows, int width, int fmt, int keep_sign, void* stream) {
    const int rc = checks("equss_ckpt_pack", x, type, ld_x, codes, ld_codes, scales, ld_scales, rows, width, fmt);
    if (rc != EQUSS_OK || rows == 0) return rc;
    Walk w;
    int64_t grid;
    if (!walk(w, rows, width, type, grid)) return equss::fail(EQUSS_E_UNSUPPORTED, "equss_ckpt_pack: %lld rows of %d channels", (long long)rows, width);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define EQUSS_PACK(T, E, K)                                                                                                       \
    hipLaunchKernelGGL((ckpt_pack_kernel<T, E, K>), dim3((unsigned)grid), dim3(kThreads), 0, s,                                   \
                       reinterpret_cast<const Elem<T>::type*>(x), ld_x, reinterpret_cast<uint8_t*>(codes), ld_codes,              \
                       reinterpret_cast<uint8_t*>(scales), ld_scales, w)
#define EQUSS_PACK_T(T)                                                                      \
    if (fmt == EQUSS_CKPT_E4M3) { if (keep_sign) EQUSS_PACK(T, true, true); else EQUSS_PACK(T, true, false); }   \
    else { if (keep_sign) EQUSS_PACK(T, false, true); else EQUSS_PACK(T, false, false); }
    if (type == EQUSS_F32) { EQUSS_PACK_T(0) }
    else if (type == EQUSS_BF16) { EQUSS_PACK_T(1) }
    else { EQUSS_PACK_T(2) }
#undef EQUSS_PACK_T
#undef EQUSS_PACK
    return equss::check_launch("ckpt_pack_kernel");
}

extern "C" int equss_ckpt_unpack(const void* codes, int64_t ld_codes, const void* scales, int64_t ld_scales, void* out, int type,
                                 int64_t ld_out, int64_t rows, int width, int fmt, void* stream) {
    const int rc = checks("equss_ckpt_unpack", out, type, ld_out, codes, ld_codes, scales, ld_scales, rows, width, fmt);
    if (rc != EQUSS_OK || rows == 0) return rc;
    Walk w;
    int64_t grid;
    if (!walk(w, rows, width, type, grid)) return equss::fail(EQUSS_E_UNSUPPORTED, "equss_ckpt_unpack: %lld rows of %d channels", (long long)rows, width);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define EQUSS_UNPACK(T, E)                                                                                                        \
    hipLaunchKernelGGL((ckpt_unpack_kernel<T, E>), dim3((unsigned)grid), dim3(kThreads), 0, s, reinterpret_cast<const uint8_t*>(codes), \
                       ld_codes, reinterpret_cast<const uint8_t*>(scales), ld_scales, reinterpret_cast<Elem<T>::type*>(out), ld_out, w)
    const bool e = fmt == EQUSS_CKPT_E4M3;
    if (type == EQUSS_F32) { if (e) EQUSS_UNPACK(0, true); else EQUSS_UNPACK(0, false); }
    else if (type == EQUSS_BF16) { if (e) EQUSS_UNPACK(1, true); else EQUSS_UNPACK(1, false); }
    else { if (e) EQUSS_UNPACK(2, true); else EQUSS_UNPACK(2, false); }
#undef EQUSS_UNPACK
    return equss::check_launch("ckpt_unpack_kernel");
}
