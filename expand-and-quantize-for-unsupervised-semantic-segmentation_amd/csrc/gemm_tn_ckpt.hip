// Weight and bias gradient of a linear layer whose input was kept in 8 bits (equss_ckpt_pack):
//     C[m][n] = sum over rows r of a[r][m] V[r][n],   bias[m] = sum over r of a[r][m],
// a (rows, M) bf16 the gradient of the layer's output, V (rows, N) the kept values; with a mask checkpoint H (rows, M), a[r][m]
// counts only where H[r][m] > 0 (the layer's output went through a ReLU whose result was kept).
//
// The summed index is the rows', the slowest of both operands, as in gemm_tn.hip: tiles lie in LDS as [row][column] and the
// fragments come out through the transposing LDS read.  The scale of a code changes from row to row, i.e. along the summed
// index, so it cannot wait for the epilogue: the codes become bf16 on their way into LDS, which is exact (ckpt.h).  The mask
// is applied to a on the same way.  The rows are split over workgroups; their partial tiles go to the workspace and a second
// kernel adds them in a fixed order, so equal calls give equal bits.
#include "ckpt.h"
#include <math.h>

namespace {

constexpr int TM = 128, TN = 128, BK = 32;
constexpr int kRowB = 256;                    // bytes per row of a tile: 128 bf16
constexpr int kTileB = BK * kRowB;
constexpr int kStageB = 2 * kTileB;
constexpr int kTnThreads = 256;

typedef uint32_t u32x4u2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4a __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

struct Args {
    const u16* a; int64_t lda;
    const uint8_t* codes; int64_t ld_codes;
    const uint8_t* scales; int64_t ld_scales;
    const uint8_t* mask; int64_t ld_mask;      // codes of H, or null
    float* c; int64_t ldc;                     // partial tiles of split s at c + s * split_c
    int64_t split_c;
    float* bias; int64_t split_bias;           // or null
    int64_t rows, rows_split;
    int M, N, tiles_m, tiles_n, splits, bias_tiles, npad, mpad;
};

// ---- the narrow form: any M (the tiled form reads 8 columns of a at once) and any leading dimensions (its offsets within a row
// range are 32 bits); 4 waves of 2 x 2 MFMA tiles, one stage ahead in registers and one in LDS
template <bool E4M3, bool MASK>
__global__ __launch_bounds__(kTnThreads, 2) void gemm_tn_ckpt_kernel(const Args g) {
    __shared__ __attribute__((aligned(16))) char smem[2 * kStageB];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles = g.tiles_m * g.tiles_n;
    const int split = blockIdx.x / tiles, tile = blockIdx.x % tiles;
    const int m0 = (tile / g.tiles_n) * TM, n0 = (tile % g.tiles_n) * TN;
    const int64_t k0 = (int64_t)split * g.rows_split;
    const int64_t k1 = k0 + g.rows_split < g.rows ? k0 + g.rows_split : g.rows;
    const int nsteps = (int)((k1 - k0 + BK - 1) / BK);

    // ---- staging: a lane moves the same 8 columns of two rows of either tile
    const int ch = tid & 15, srow = tid >> 4;
    const int ma = m0 + 8 * ch, nb = n0 + 8 * ch;
    const bool a_whole = ma + 8 <= g.M, a_any = ma < g.M, b_any = nb < g.npad;
    u32x4a ra[2];
    uint2 rb[2], rm[2];
    uint32_t rs[2];
    auto load = [&](int step) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t r = k0 + (int64_t)step * BK + srow + 16 * i;
            const bool in = r < k1;
            ra[i] = u32x4a{0, 0, 0, 0};
            rb[i] = rm[i] = make_uint2(0, 0);
            rs[i] = 0;
            if (in && a_whole) {
                const u32x4u2 v = *reinterpret_cast<const u32x4u2*>(g.a + r * g.lda + ma);
                ra[i] = u32x4a{v[0], v[1], v[2], v[3]};
            } else if (in && a_any) {
                const u16* p = g.a + r * g.lda + ma;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (ma + j < g.M) ra[i][j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
            }
            if (MASK && in && a_any) rm[i] = *reinterpret_cast<const uint2*>(g.mask + r * g.ld_mask + ma);
            if (in && b_any) {
                rb[i] = *reinterpret_cast<const uint2*>(g.codes + r * g.ld_codes + nb);
                rs[i] = g.scales[r * g.ld_scales + nb / equss::kCkptBlock];
            }
        }
    };
    float bsum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) bsum[j] = 0.f;
    const bool want_bias = g.bias != nullptr && n0 == 0;
    auto store = [&](int buf) {
        char* sb = smem + buf * kStageB;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = srow + 16 * i;
            if constexpr (MASK) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t w = (j & 2 ? rm[i].y : rm[i].x) >> (16 * (j & 1));
                    const uint32_t keep = ((int8_t)w > 0 ? 0xffffu : 0u) | ((int8_t)(w >> 8) > 0 ? 0xffff0000u : 0u);
                    ra[i][j] &= keep;
                }
            }
            if (want_bias) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    bsum[2 * j] += equss::bits_as<float>(ra[i][j] << 16);
                    bsum[2 * j + 1] += equss::bits_as<float>(ra[i][j] & 0xffff0000u);
                }
            }
            const int at = r * kRowB + ((ch ^ (4 * (r & 3))) * 16);
            *reinterpret_cast<u32x4a*>(sb + at) = ra[i];
            const float s = equss::ckpt_scale(rs[i]);
            const f32x4 lo = equss::ckpt_decode4<E4M3>(rb[i].x), hi = equss::ckpt_decode4<E4M3>(rb[i].y);
            *reinterpret_cast<u32x4a*>(sb + kTileB + at) =
                u32x4a{equss::pack_bf16(lo[0] * s, lo[1] * s), equss::pack_bf16(lo[2] * s, lo[3] * s),
                       equss::pack_bf16(hi[0] * s, hi[1] * s), equss::pack_bf16(hi[2] * s, hi[3] * s)};
        }
    };

    // ---- fragment reads: wave tile 64 x 64 = 2 x 2 MFMA tiles; a 16-lane group reads a 4 (row) x 16 (column) block, every lane
    // gets one column of it
    const int wm = wave >> 1, wn = wave & 1;
    const int q = (lane >> 2) & 3, pp = lane & 3, hg = (lane >> 4) & 1, kb = lane >> 5;
    auto frag_at = [&](int c0) {
        const int chunk = c0 / 8 + 2 * hg + (pp >> 1);
        return (8 * kb + q) * kRowB + ((chunk ^ (4 * q)) * 16) + (pp & 1) * 8;
    };
    auto frag = [&](int at) {
        typedef __attribute__((address_space(3))) i16x4* lds_p;
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(smem + at));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(smem + at + 4 * kRowB));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    if (nsteps > 0) {
        load(0);
        store(0);
    }
    __syncthreads();
    for (int step = 0; step < nsteps; ++step) {
        const int buf = step & 1;
        if (step + 1 < nsteps) load(step + 1);
#pragma unroll
        for (int ks = 0; ks < BK / 16; ++ks) {
            const int base = buf * kStageB + ks * 16 * kRowB;
            bf16x8 af[2], bf[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                af[t] = frag(base + frag_at(wm * 64 + t * 32));
                bf[t] = frag(base + kTileB + frag_at(wn * 64 + t * 32));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[i], bf[j], acc[i][j], 0, 0, 0);
        }
        if (step + 1 < nsteps) store(buf ^ 1);
        __syncthreads();
    }

    // register r of an accumulator is row (r & 3) + 8 (r >> 2) + 4 kb of the 32 x 32 tile, lane & 31 its column
    float* c = g.c + split * g.split_c;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = n0 + wn * 64 + j * 32 + (lane & 31);
            if (n < g.N) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int m = m0 + wm * 64 + i * 32 + 4 * kb + (r & 3) + 8 * (r >> 2);
                    if (m < g.M) c[m * g.ldc + n] = acc[i][j][r];
                }
            }
        }
    if (want_bias) {
        float* part = reinterpret_cast<float*>(smem);      // (the last barrier of the loop is behind every reader of the tiles)
#pragma unroll
        for (int j = 0; j < 8; ++j) part[srow * TM + 8 * ch + j] = bsum[j];
        __syncthreads();
        if (tid < TM && m0 + tid < g.M) {
            float s = 0.f;
            for (int r = 0; r < kTnThreads / 16; ++r) s += part[r * TM + tid];
            g.bias[split * g.split_bias + m0 + tid] = s;
        }
    }
}

// ---- square tiles of TILE = 256 (8 waves, two a SIMD, one workgroup a CU) or 128 (4 waves, two workgroups a CU) of C, in
// 2 x TILE / 64 waves of TILE / 64 x 2 MFMA tiles of 32 x 32; 32 rows a stage, four stages in LDS.
// While a stage's fragments are multiplied,
//   the fragments of the next half stage are read (the next stage's first half too: its writes are a barrier back),
//   the stage after the next goes from registers through the conversion into its slot of LDS, and
//   each of those registers is requested again from two stages further on (there are two sets of them: one stage of 32 rows
//   takes half a microsecond, less than a load from memory does under load),
// without a branch in between, so that the scheduler can put all of it between the MFMAs.  The loop goes by four stages, so that
// slots and register sets are constants.  Loads past a workgroup's rows return zero (buffer addressing), codes and scales too:
// the last stages need no care and the surplus ones of the last round multiply zeros.
// Conversions, address arithmetic and the bias are what the matrix pipe waits for; hence two waves a SIMD, constant LDS addresses
// and buffer loads.  Counted at 102400 rows, 1024 x 768, int8: 5.0 million MFMAs hold the matrix pipes for 54 % of the launch,
// beside 22 million other vector instructions; 327 MB read, 69 written.
// 102400 rows, 1024 x 768, bias and join included: int8 165 us, e4m3 (whose conversion is one instruction for two values) 160 us,
// 0.98 and 1.01 PFLOP/s; an 8192^3 bf16 library product runs at 1.25.  Another 102400 rows add 130 and 128 us (1.24 and 1.26
// PFLOP/s); what does not grow with the rows, the partial products (256 KB a CU) and their join among it, is 30 to 40 us.
// Consecutive row ranges and tiles on one XCD: 175 us, 184 dealt round (102400 rows, 384 x 384: 55 / 70).  The large tile spills
// a few registers, 24 bytes a lane; two of them are read back in each stage of the int8 form.
// Columns past M: the last chunk of 8 columns is read at M - 8, so that every load is whole and inside; its columns then
// overlap the chunk before, both give the same sums, and both are written.  Columns past N lie in the checkpoint's padding or
// are read from its last block; their sums are dropped.
constexpr int kBigBK = 32, kSlots = 4;

template <bool E4M3>
__device__ __forceinline__ u32x4a to_bf16x8(uint32_t c0, uint32_t c1, float s) {
    if constexpr (E4M3) {
        typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
        const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c0, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c0, s, true);
        const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c1, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c1, s, true);
        return u32x4a{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)};
    } else {
        const f32x4 lo = equss::ckpt_decode4<false>(c0), hi = equss::ckpt_decode4<false>(c1);
        return u32x4a{equss::pack_bf16(lo[0] * s, lo[1] * s), equss::pack_bf16(lo[2] * s, lo[3] * s),
                      equss::pack_bf16(hi[0] * s, hi[1] * s), equss::pack_bf16(hi[2] * s, hi[3] * s)};
    }
}

// rows [row0, row0 + rows) of a matrix of `ld` bytes a row: loads past the end return zero
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* p, int64_t ld, int64_t row0, int rows) {
    const uint64_t base = reinterpret_cast<uint64_t>(p) + (uint64_t)row0 * (uint64_t)ld;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)base), hi = __builtin_amdgcn_readfirstlane((uint32_t)(base >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0,
                                             __builtin_amdgcn_readfirstlane((int)((int64_t)rows * ld)), 0x00020000);
}

template <bool E4M3, bool MASK, int TILE>
__global__ __launch_bounds__(2 * TILE, 2) void gemm_tn_ckpt_tile_kernel(const Args g) {
    constexpr int THREADS = 2 * TILE, WAVES_N = TILE / 64, WM = TILE / 64, WNW = 2;
    constexpr int TMB = TILE, TNB = TILE, RA = 2 * TILE, RB = 2 * TILE, SLOT = kBigBK * (RA + RB);
    constexpr int ACH = TILE / 8, BCH = TILE / 16;          // a row's chunks of 8 columns of a, of 16 codes
    constexpr int AP = kBigBK * ACH / THREADS, BP = kBigBK * BCH / THREADS;   // passes of the threads over a stage: 2 and 1
    constexpr int AROWS = THREADS / ACH, BROWS = THREADS / BCH;               // rows a pass
    static_assert(AP == 2 && BP == 1, "one request of a a half stage, one of the codes a stage");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles = g.tiles_m * g.tiles_n, total = tiles * g.splits;
    // consecutive units on one XCD (workgroups go round the eight of them): the tiles of a row range share its L2
    const int per = (total + 7) / 8, unit = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if ((int)(blockIdx.x / 8) >= per || unit >= total) return;
    const int split = unit / tiles, tile = unit % tiles;
    const int m0 = (tile / g.tiles_n) * TMB, tn = tile % g.tiles_n, n0 = tn * TNB;
    const int64_t k0 = (int64_t)split * g.rows_split;
    const int64_t k1 = k0 + g.rows_split < g.rows ? k0 + g.rows_split : g.rows;
    const int rows = k1 > k0 ? (int)(k1 - k0) : 0;
    const int stages = (rows + kBigBK - 1) / kBigBK;

    // ---- staging
    const int ach = tid % ACH, arow = tid / ACH, bch = tid % BCH, brow = tid / BCH;
    int ma = m0 + 8 * ach, nb = n0 + 16 * bch;
    ma = ma + 8 <= g.M ? ma : g.M - 8;
    nb = nb + 16 <= g.npad ? nb : g.npad - 16;
    const __amdgpu_buffer_rsrc_t a_rs = rows_rsrc(g.a, g.lda * 2, k0, rows), b_rs = rows_rsrc(g.codes, g.ld_codes, k0, rows);
    const __amdgpu_buffer_rsrc_t s_rs = rows_rsrc(g.scales, g.ld_scales, k0, rows), m_rs = rows_rsrc(g.mask, g.ld_mask, k0, MASK ? rows : 0);
    // byte offsets of the next request of every pass
    uint32_t va[AP], vm[AP], vb[BP], vs[BP];
#pragma unroll
    for (int i = 0; i < AP; ++i) {
        va[i] = (uint32_t)(((arow + AROWS * i) * (int)g.lda + ma) * 2);
        vm[i] = (uint32_t)((arow + AROWS * i) * (int)g.ld_mask + ma);
    }
#pragma unroll
    for (int i = 0; i < BP; ++i) {
        vb[i] = (uint32_t)((brow + BROWS * i) * (int)g.ld_codes + nb);
        vs[i] = (uint32_t)((brow + BROWS * i) * (int)g.ld_scales + nb / equss::kCkptBlock);
    }
    const uint32_t da = (uint32_t)(kBigBK * 2 * (int)g.lda), dm = (uint32_t)(kBigBK * (int)g.ld_mask);
    const uint32_t db = (uint32_t)(kBigBK * (int)g.ld_codes), ds = (uint32_t)(kBigBK * (int)g.ld_scales);
    u32x4a ra[2][AP], rb[2][BP];
    uint2 rm[2][AP];
    uint32_t rs[2][BP];
    auto load_a = [&](int set, int i) __attribute__((always_inline)) {
        ra[set][i] = __builtin_amdgcn_raw_buffer_load_b128(a_rs, va[i], 0, 0);
        va[i] += da;
        if constexpr (MASK) {
            typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
            const u32x2v c = __builtin_amdgcn_raw_buffer_load_b64(m_rs, vm[i], 0, 0);
            rm[set][i] = make_uint2(c[0], c[1]);
            vm[i] += dm;
        }
    };
    auto load_b = [&](int set, int i) __attribute__((always_inline)) {
        rb[set][i] = __builtin_amdgcn_raw_buffer_load_b128(b_rs, vb[i], 0, 0);
        rs[set][i] = __builtin_amdgcn_raw_buffer_load_b8(s_rs, vs[i], 0, 0);
        vb[i] += db;
        vs[i] += ds;
    };
    float bsum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) bsum[j] = 0.f;
    char* const wa = smem + arow * RA + ((ach ^ (4 * (arow & 3))) * 16);                 // (AROWS and BROWS are multiples of 4)
    char* const wb0 = smem + kBigBK * RA + brow * RB + (((2 * bch) ^ (4 * (brow & 3))) * 16);
    char* const wb1 = smem + kBigBK * RA + brow * RB + (((2 * bch + 1) ^ (4 * (brow & 3))) * 16);
    auto store_a = [&](auto bias_c, int set, int i, int slot) __attribute__((always_inline)) {
        u32x4a v = ra[set][i];
        if constexpr (MASK) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w = (j & 2 ? rm[set][i].y : rm[set][i].x) >> (16 * (j & 1));
                v[j] &= ((int8_t)w > 0 ? 0xffffu : 0u) | ((int8_t)(w >> 8) > 0 ? 0xffff0000u : 0u);
            }
        }
        if constexpr (decltype(bias_c)::value) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                bsum[2 * j] += equss::bits_as<float>(v[j] << 16);
                bsum[2 * j + 1] += equss::bits_as<float>(v[j] & 0xffff0000u);
            }
        }
        *reinterpret_cast<u32x4a*>(wa + slot * SLOT + i * AROWS * RA) = v;
    };
    auto store_b = [&](int set, int i, int slot) __attribute__((always_inline)) {
        const u32x4a c = rb[set][i];
        const float s = equss::ckpt_scale(rs[set][i]);
        *reinterpret_cast<u32x4a*>(wb0 + slot * SLOT + i * BROWS * RB) = to_bf16x8<E4M3>(c[0], c[1], s);
        *reinterpret_cast<u32x4a*>(wb1 + slot * SLOT + i * BROWS * RB) = to_bf16x8<E4M3>(c[2], c[3], s);
    };

    const int wm = wave / WAVES_N, wn = wave % WAVES_N;
    const int q = (lane >> 2) & 3, pp = lane & 3, hg = (lane >> 4) & 1, kb = lane >> 5;
    auto frag_at = [&](int c0, int row_bytes) __attribute__((always_inline)) {
        const int chunk = c0 / 8 + 2 * hg + (pp >> 1);
        return (8 * kb + q) * row_bytes + ((chunk ^ (4 * q)) * 16) + (pp & 1) * 8;
    };
    typedef __attribute__((address_space(3))) i16x4* lds_p;
    auto frag = [&](const char* at, int row_bytes) __attribute__((always_inline)) {
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(at));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(at + 4 * row_bytes));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    const char *a_at[WM], *b_at[WNW];
#pragma unroll
    for (int t = 0; t < WM; ++t) a_at[t] = smem + frag_at((wm * WM + t) * 32, RA);
#pragma unroll
    for (int t = 0; t < WNW; ++t) b_at[t] = smem + kBigBK * RA + frag_at((wn * WNW + t) * 32, RB);
    bf16x8 af[2][WM], bf[2][WNW];
    auto read = [&](int set, int slot, int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < WNW; ++t) bf[set][t] = frag(b_at[t] + slot * SLOT + ks * 16 * RB, RB);
#pragma unroll
        for (int t = 0; t < WM; ++t) af[set][t] = frag(a_at[t] + slot * SLOT + ks * 16 * RA, RA);
    };
    f32x16 acc[WM][WNW];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WNW; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    auto multiply = [&](int set) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < WM; ++i)
#pragma unroll
            for (int j = 0; j < WNW; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[set][i], bf[set][j], acc[i][j], 0, 0, 0);
    };
    using No = std::false_type;
    using Yes = std::true_type;
    // one stage: multiply slot S, read ahead, store the stage after the next (register set S & 1) and request the one two behind it
    auto step = [&](auto bias_c, auto slot_c) __attribute__((always_inline)) {
        constexpr int S = decltype(slot_c)::value, SET = S & 1, S1 = (S + 1) & 3, S2 = (S + 2) & 3;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (ks == 0) read(1, S, 1);
            else read(0, S1, 0);
#pragma unroll
            for (int i = ks * AP / 2; i < (ks + 1) * AP / 2; ++i) { store_a(bias_c, SET, i, S2); load_a(SET, i); }
#pragma unroll
            for (int i = ks == 0 ? 0 : BP; i < BP; ++i) { store_b(SET, i, S2); load_b(SET, i); }
            multiply(ks);
            // the order wanted: behind every MFMA some fragment reads, conversions, and further on the stores and requests.  Three
            // reads against two (102400 rows, us): int8 1024 x 768 169 / 172, 384 x 384 52 / 54, e4m3 384 x 384 49 / 50; two in
            // the large e4m3 tile, which is short of registers: 1024 x 768 160 / 172
            constexpr int READS = E4M3 && TILE == 256 ? 2 : 3;
#pragma unroll
            for (int i = 0; i < WM * WNW; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);            // MFMA
                if (i * READS < 2 * (WM + WNW)) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);   // LDS reads
                __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);            // VALU
                if (i >= WM * WNW / 2) {
                    __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);        // LDS write
                    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);        // global load
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
    };
    // the bias: each of the first `bias_tiles` tiles of a row of tiles adds up its share of the stages, [bias0, bias1); whole
    // rounds of four
    const int rounds = (stages + 3) / 4;
    const bool adds = g.bias && tn < g.bias_tiles;
    const int bias0 = adds ? (int)((int64_t)rounds * tn / g.bias_tiles) : 0;
    const int bias1 = adds ? (int)((int64_t)rounds * (tn + 1) / g.bias_tiles) : 0;
    {
        // stages 0 and 1 into their slots, 2 and 3 requested
        auto first = [&](auto bias_c) __attribute__((always_inline)) {
#pragma unroll
            for (int set = 0; set < 2; ++set) {
#pragma unroll
                for (int i = 0; i < AP; ++i) store_a(bias_c, set, i, set);
#pragma unroll
                for (int i = 0; i < BP; ++i) store_b(set, i, set);
            }
        };
#pragma unroll
        for (int set = 0; set < 2; ++set) {
#pragma unroll
            for (int i = 0; i < AP; ++i) load_a(set, i);
#pragma unroll
            for (int i = 0; i < BP; ++i) load_b(set, i);
        }
        if (bias0 == 0 && bias1 > 0) first(Yes());
        else first(No());
#pragma unroll
        for (int set = 0; set < 2; ++set) {
#pragma unroll
            for (int i = 0; i < AP; ++i) load_a(set, i);
#pragma unroll
            for (int i = 0; i < BP; ++i) load_b(set, i);
        }
    }
    __syncthreads();
    read(0, 0, 0);
    // A round stores stages 2 .. 5 of its own count, so the stores of [4 bias0, 4 bias1) are: the second half of round bias0 - 1
    // (the start above for 0), the rounds from bias0 on, and the first half of round bias1 - 1.
    using S0 = std::integral_constant<int, 0>;
    using S1c = std::integral_constant<int, 1>;
    using S2c = std::integral_constant<int, 2>;
    using S3c = std::integral_constant<int, 3>;
    int round = 0;
    auto run = [&](auto first_half, auto second_half, int to) __attribute__((always_inline)) {
        for (; round < to; ++round) {
            step(first_half, S0());
            step(first_half, S1c());
            step(second_half, S2c());
            step(second_half, S3c());
        }
    };
    if (stages <= 2) {                                      // both are in LDS and counted: half a round
        for (; round < rounds; ++round) {
            step(No(), S0());
            step(No(), S1c());
        }
    }
    if (adds) {
        run(No(), No(), bias0 - 1);
        if (bias1 > bias0) {
            run(No(), Yes(), bias0);
            run(Yes(), Yes(), bias1 - 1);
            run(Yes(), No(), bias1);
        }
    }
    run(No(), No(), rounds);

    float* c = g.c + split * g.split_c;
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int chunk = m0 + (wm * WM + i) * 32 + 8 * (r >> 2);
            if (chunk < g.M) {
                const int m = (chunk + 8 <= g.M ? chunk : g.M - 8) + 4 * kb + (r & 3);
#pragma unroll
                for (int j = 0; j < WNW; ++j) {
                    const int n = n0 + (wn * WNW + j) * 32 + (lane & 31);
                    if (n < g.N) c[m * g.ldc + n] = acc[i][j][r];
                }
            }
        }
    if (adds) {
        float* part = reinterpret_cast<float*>(smem);      // (every reader of the tiles is behind the loop's last barrier)
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) part[arow * (8 * ACH) + 8 * ach + j] = bsum[j];
        __syncthreads();
        const int chunk = m0 + tid / 8 * 8;
        if (tid < TMB && chunk < g.M) {
            float s = 0.f;
            for (int r = 0; r < AROWS; ++r) s += part[r * (8 * ACH) + tid];
            g.bias[(split * g.bias_tiles + tn) * g.split_bias + (chunk + 8 <= g.M ? chunk : g.M - 8) + tid % 8] = s;
        }
    }
}

// C = sum of the partial products, in the order of the splits; then the bias
__global__ __launch_bounds__(256) void gemm_tn_join_kernel(const float* __restrict__ part, int64_t split_c, float* __restrict__ c,
                                                          int64_t ldc, const float* __restrict__ bpart, int64_t split_bias,
                                                          float* __restrict__ bias, int splits, int bias_splits, int M, int N) {
    const int64_t cells = (int64_t)M * N;
    const int64_t total = cells + (bias ? M : 0);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const bool main = i < cells;
        const float* p = main ? part + i : bpart + (i - cells);
        const int64_t step = main ? split_c : split_bias;
        const int n = main ? splits : bias_splits;
        float s = 0.f;
        for (int k = 0; k < n; k += 16) {                  // (sixteen loads in flight: one row range is a load, and they add up)
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = p[(k + j < n ? k + j : n - 1) * step];
#pragma unroll
            for (int j = 0; j < 16; ++j) s += k + j < n ? v[j] : 0.f;
        }
        if (main) c[(i / N) * ldc + i % N] = s;
        else bias[i - cells] = s;
    }
}

struct Plan { int tile, tiles_m, tiles_n, splits, bias_splits; int64_t rows_split; };

// 32-bit byte offsets within a workgroup's rows (and the stages that the loop asks for behind them, eight at most)
bool offsets_fit(const Plan& p, int64_t ld_bytes) { return (p.rows_split + 16 * kBigBK) * ld_bytes < ((int64_t)1 << 31); }

// tile 0: the narrow kernel (tiles of TM x TN)
Plan plan(int64_t rows, int M, int N, int tile) {
    Plan p;
    p.tile = tile;
    const int t = tile ? tile : TM, bk = BK;
    p.tiles_m = (M + t - 1) / t;
    p.tiles_n = (N + t - 1) / t;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    // Row ranges: more of them shorten everybody's loop (32 rows take 0.35 us, 0.75 us with the large tile and all CUs at work),
    // but two or more need the join (6 us for its launch and what it waits for), and each writes and reads back a partial product
    // (0.08 us + 1.1 us for a million elements).  The cheapest number, at least four steps each, at most one round of workgroups;
    // one where that is cheaper (512 rows, 1024 x 768: 11.5 us, 16.7 with two ranges).
    const int64_t steps = (rows + bk - 1) / bk, round = (tile == 256 ? 256 : 512) / tiles;
    const double step = tile == 256 ? 0.75 : 0.35, range = 0.08 + 1.1e-6 * M * N;
    int64_t splits = (int64_t)(sqrt((double)steps * step / range) + 0.5);
    if (splits > round) splits = round;
    if (splits > steps / 4) splits = steps / 4;
    if (splits <= 1 || (double)(steps - steps / splits) * step < 6.0 + (double)splits * range) splits = 1;
    p.rows_split = ((rows + splits - 1) / splits + bk - 1) / bk * bk;
    if (p.rows_split < bk) p.rows_split = bk;
    p.splits = (int)((rows + p.rows_split - 1) / p.rows_split);
    if (p.splits < 1) p.splits = 1;
    // (one row range: the first tile of a row of tiles adds all of the bias, and there is nothing to join)
    p.bias_splits = tile && p.splits > 1 ? p.splits * p.tiles_n : p.splits;
    return p;
}

// The large tile reads half as much LDS for a product, which pays where every CU has a long way to go (2e10 products) and little of
// the tile lies outside: more than three small tiles to a large one.  Measured (us, int8; 128 against 256):
//   25088 x 1024 x 768 60 / 63, 51200 x 1024 x 768 102 / 92, 102400 x 1024 x 768 204 / 169, 102400 x 512 x 512 77 / 73
//   three to one: 102400 x 1024 x 384 113 / 113, 102400 x 384 x 768 85 / 90;  fewer: 640 x 384 72 / 85, 384 x 384 52 / 62
// Through a mask it runs out of registers: 102400 rows, 768 x 768 188 / 194, 640 x 384 90 / 118, 384 x 384 59 / 82, 1024 x 768
// 247 / 242, and only long and narrow products would gain (1024 x 200 104 / 92); it has no such form.
int tile_of(int64_t rows, int M, int N, bool mask) {
    if (M < 8) return 0;
    const int64_t small = (int64_t)((M + 127) / 128) * ((N + 127) / 128), large = (int64_t)((M + 255) / 256) * ((N + 255) / 256);
    return !mask && (double)rows * M * N >= 2e10 && small > 3 * large ? 256 : 128;
}

constexpr int kMostCols = 1 << 30;     // columns are 32-bit numbers, and rounded up

// partial products and, behind them, partial bias sums; nothing where one row range writes the results
size_t workspace(const Plan& p, int M, int N) {
    return p.splits == 1 ? 0 : ((size_t)p.splits * M * N + (size_t)p.bias_splits * M) * sizeof(float);
}

}  // namespace

extern "C" size_t equss_gemm_tn_ckpt_workspace_bytes(int64_t rows, int M, int N) {
    if (rows < 0 || M <= 0 || N <= 0 || M > kMostCols || N > kMostCols) return 0;
    // with a mask or without, and the narrow kernel, which stands in where leading dimensions are too long for the others
    const int tiles[3] = {tile_of(rows, M, N, false), tile_of(rows, M, N, true), 0};
    size_t most = 0;
    for (int tile : tiles) {
        const size_t one = workspace(plan(rows, M, N, tile), M, N);
        if (one > most) most = one;
    }
    return most;
}

extern "C" int equss_gemm_tn_ckpt(const void* a, int64_t lda, const void* codes, int64_t ld_codes, const void* scales, int64_t ld_scales,
                                  int fmt, const void* relu_codes, int64_t ld_relu, float* C, int64_t ldc, float* bias, int64_t rows,
                                  int M, int N, void* workspace_ptr, size_t workspace_bytes, void* stream) {
    if (rows < 0 || M <= 0 || N <= 0) return equss::fail(EQUSS_E_SHAPE, "equss_gemm_tn_ckpt: rows=%lld M=%d N=%d", (long long)rows, M, N);
    if (M > kMostCols || N > kMostCols) return equss::fail(EQUSS_E_UNSUPPORTED, "equss_gemm_tn_ckpt: M=%d N=%d (at most %d)", M, N, kMostCols);
    if (fmt != EQUSS_CKPT_INT8 && fmt != EQUSS_CKPT_E4M3) return equss::fail(EQUSS_E_UNSUPPORTED, "equss_gemm_tn_ckpt: format %d", fmt);
    if (!C || (rows > 0 && (!a || !codes || !scales))) return equss::fail(EQUSS_E_NULL, "equss_gemm_tn_ckpt: null pointer argument");
    Args g;
    g.npad = (N + equss::kCkptBlock - 1) / equss::kCkptBlock * equss::kCkptBlock;
    g.mpad = (M + equss::kCkptBlock - 1) / equss::kCkptBlock * equss::kCkptBlock;
    if (ldc < N || (rows > 0 && (lda < M || ld_codes < g.npad || (ld_codes % equss::kCkptBlock) != 0 || ((uintptr_t)codes % 16) != 0 ||
                                 ld_scales < g.npad / equss::kCkptBlock || ((uintptr_t)a % 2) != 0)))
        return equss::fail(EQUSS_E_ALIGN, "equss_gemm_tn_ckpt: codes 16-byte aligned with a leading dimension that is a multiple of 32 and "
                           "holds %d, rows of %d and %d elements", g.npad, M, N);
    if (rows > 0 && relu_codes && (ld_relu < g.mpad || (ld_relu % equss::kCkptBlock) != 0 || ((uintptr_t)relu_codes % 16) != 0))
        return equss::fail(EQUSS_E_ALIGN, "equss_gemm_tn_ckpt: mask codes 16-byte aligned with a leading dimension that is a multiple of 32 "
                           "and holds %d", g.mpad);
    const size_t need = equss_gemm_tn_ckpt_workspace_bytes(rows, M, N);
    Plan p = plan(rows, M, N, tile_of(rows, M, N, relu_codes != nullptr));
    if (p.tile && !(offsets_fit(p, lda * 2) && offsets_fit(p, ld_codes) && offsets_fit(p, ld_scales) && offsets_fit(p, relu_codes ? ld_relu : 0)))
        p = plan(rows, M, N, 0);
    if (need > 0 && (!workspace_ptr || workspace_bytes < need || ((uintptr_t)workspace_ptr % 16) != 0))
        return equss::fail(EQUSS_E_WORKSPACE, "equss_gemm_tn_ckpt: workspace of %zu bytes, 16-byte aligned, needed", need);
    const int64_t blocks = (int64_t)p.tiles_m * p.tiles_n * p.splits;
    if (blocks + 7 > equss::max_blocks(2 * 256) || (p.rows_split + BK - 1) / BK > 0x7fffffff)
        return equss::fail(EQUSS_E_UNSUPPORTED, "equss_gemm_tn_ckpt: %lld rows, M=%d N=%d", (long long)rows, M, N);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    g.a = reinterpret_cast<const u16*>(a); g.lda = lda;
    g.codes = reinterpret_cast<const uint8_t*>(codes); g.ld_codes = ld_codes;
    g.scales = reinterpret_cast<const uint8_t*>(scales); g.ld_scales = ld_scales;
    g.mask = reinterpret_cast<const uint8_t*>(relu_codes); g.ld_mask = ld_relu;
    g.rows = rows; g.rows_split = p.rows_split; g.M = M; g.N = N; g.tiles_m = p.tiles_m; g.tiles_n = p.tiles_n; g.splits = p.splits; g.bias_tiles = p.bias_splits / p.splits;
    float* part = reinterpret_cast<float*>(workspace_ptr);
    float* bpart = part + (size_t)p.splits * M * N;
    const bool direct = p.splits == 1;
    g.c = direct ? C : part; g.ldc = direct ? ldc : N; g.split_c = direct ? 0 : (int64_t)M * N;
    g.bias = bias ? (direct ? bias : bpart) : nullptr; g.split_bias = M;
    const bool e = fmt == EQUSS_CKPT_E4M3;
    if (p.tile) {
        const dim3 grid((unsigned)((blocks + 7) / 8 * 8));
        const int lds = kSlots * kBigBK * 4 * p.tile;
#define EQUSS_TN_TILE(E, K, T)                                                                                                 \
    do {                                                                                                                       \
        if (!equss::lds_opt_in(reinterpret_cast<const void*>(&gemm_tn_ckpt_tile_kernel<E, K, T>), lds))                        \
            return equss::fail(EQUSS_E_UNSUPPORTED, "equss_gemm_tn_ckpt: %d bytes of LDS", lds);                               \
        hipLaunchKernelGGL((gemm_tn_ckpt_tile_kernel<E, K, T>), grid, dim3(2 * T), lds, s, g);                                 \
    } while (0)
        if (p.tile == 256) { if (e) EQUSS_TN_TILE(true, false, 256); else EQUSS_TN_TILE(false, false, 256); }
        else if (relu_codes) { if (e) EQUSS_TN_TILE(true, true, 128); else EQUSS_TN_TILE(false, true, 128); }
        else { if (e) EQUSS_TN_TILE(true, false, 128); else EQUSS_TN_TILE(false, false, 128); }
#undef EQUSS_TN_TILE
    } else {
        const dim3 grid((unsigned)blocks), block(kTnThreads);
        if (e) {
            if (relu_codes) hipLaunchKernelGGL((gemm_tn_ckpt_kernel<true, true>), grid, block, 0, s, g);
            else hipLaunchKernelGGL((gemm_tn_ckpt_kernel<true, false>), grid, block, 0, s, g);
        } else {
            if (relu_codes) hipLaunchKernelGGL((gemm_tn_ckpt_kernel<false, true>), grid, block, 0, s, g);
            else hipLaunchKernelGGL((gemm_tn_ckpt_kernel<false, false>), grid, block, 0, s, g);
        }
    }
    const int rc = equss::check_launch("gemm_tn_ckpt_kernel");
    if (rc != EQUSS_OK || direct) return rc;
    const int64_t join = (int64_t)M * N + (bias ? M : 0);
    int64_t gx = (join + 255) / 256;
    if (gx > 4096) gx = 4096;
    hipLaunchKernelGGL(gemm_tn_join_kernel, dim3((unsigned)gx), dim3(256), 0, s, part, (int64_t)M * N, C, ldc, bpart, (int64_t)M, bias, p.splits,
                       p.bias_splits, M, N);
    return equss::check_launch("gemm_tn_join_kernel");
}
