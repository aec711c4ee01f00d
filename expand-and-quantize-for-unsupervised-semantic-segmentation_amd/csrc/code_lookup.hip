// Codewords by their indices, with a scale, and the gradient of that lookup.
//   equss_code_lookup:       out[r][p d + j] = scale * books[p][idx[p][r]][j], 0 where the index lies outside [0, K)
//   equss_code_lookup_grad:  g_books[p][k][j] = scale * sum over r with idx[p][r] = k of g[r][p d + j]
// The lookup writes its output once and reads the codebooks out of L2 (1 MB for 8 x 256 x 128 in fp32): it is bound by the
// stores.  A lane owns 16 bytes of the output.  102400 rows, 8 x 256 x 128: bf16 39 us (5.3 TB/s of 211 MB), fp32 79 us (5.3 TB/s;
// 86 with stores through the caches).  The gradient walks the rows in the order of their codes: code_sort.h.  Of the same rows in
// fp32 it takes 96 us: 72 in the walk (5.9 TB/s of 419 MB), 18 in the sort, 6.3 in the join.
#include "code_sort.h"

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2u2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4u2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));

template <int T> struct Elem;    // 0 fp32, 1 bf16, 2 fp16
template <> struct Elem<0> { typedef float type; };
template <> struct Elem<1> { typedef u16 type; };
template <> struct Elem<2> { typedef _Float16 type; };

template <int T>
__device__ __forceinline__ float to_f32(typename Elem<T>::type v) {
    if constexpr (T == 1) return equss::bf2f(v);
    else return (float)v;
}
template <int T>
__device__ __forceinline__ typename Elem<T>::type from_f32(float v) {
    if constexpr (T == 1) return equss::f2bf(v);
    else return (typename Elem<T>::type)v;
}
template <int T>
__device__ __forceinline__ uint32_t scaled_pair(uint32_t w, float scale) {
    if constexpr (T == 1)
        return equss::pack_bf16(__builtin_bit_cast(float, w << 16) * scale, __builtin_bit_cast(float, w & 0xffff0000u) * scale);
    else {
        const f16x2v h = __builtin_bit_cast(f16x2v, w);
        return __builtin_bit_cast(uint32_t, f16x2v{(_Float16)((float)h.x * scale), (_Float16)((float)h.y * scale)});
    }
}

struct LookupArgs {
    equss::IndexView index;
    const void* books;
    void* out; int64_t ld_out;
    int64_t rows;
    float scale;
    int num_pq, d, width, units_row, units_code, rows_wg;
    uint32_t K, magic_row, magic_code;      // ceil(2^32 / units); 0 where units is 1
};

__device__ __forceinline__ uint32_t divide(uint32_t a, uint32_t magic, uint32_t by_one) { return by_one ? a : __umulhi(a, magic); }

// WHOLE: a code's d elements are whole 16-byte units (fewer than 65536 of them) and rows start on 16 bytes; otherwise a unit is gathered element by element
// and stored at whatever address it has.
template <int T, bool WHOLE>
__global__ __launch_bounds__(256) void code_lookup_kernel(const LookupArgs a) {
    constexpr int V = T == 0 ? 4 : 8;
    typedef typename Elem<T>::type E;
    const int64_t row0 = (int64_t)blockIdx.x * a.rows_wg, left = a.rows - row0;
    const uint32_t units = (uint32_t)((left < a.rows_wg ? left : a.rows_wg) * a.units_row);
    const E* books = reinterpret_cast<const E*>(a.books);
    for (uint32_t u = threadIdx.x; u < units; u += 256) {
        const uint32_t lr = a.rows_wg == 1 ? 0u : divide(u, a.magic_row, a.units_row == 1);
        const uint32_t c = u - lr * (uint32_t)a.units_row;
        const int64_t r = row0 + lr;
        E* dst = reinterpret_cast<E*>(a.out) + r * a.ld_out + (int64_t)c * V;
        if constexpr (WHOLE) {
            const uint32_t p = divide(c, a.magic_code, a.units_code == 1);
            const uint32_t k = equss::code_at(a.index, (int)p, r, a.K);
            u32x4v w = {0, 0, 0, 0};
            if (k != a.K) {
                w = *reinterpret_cast<const u32x4v*>(books + ((int64_t)p * a.K + k) * a.d + (int64_t)(c - p * a.units_code) * V);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = T == 0 ? __builtin_bit_cast(uint32_t, equss::bits_as<float>(w[i]) * a.scale) : scaled_pair<T == 0 ? 1 : T>(w[i], a.scale);
            }
            __builtin_nontemporal_store(w, reinterpret_cast<u32x4v*>(dst));
        } else {
            int col = (int)c * V;
            uint32_t p = (uint32_t)col / (uint32_t)a.d;
            int j = col - (int)p * a.d;
            uint32_t k = equss::code_at(a.index, (int)p, r, a.K);
            E v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[i] = (E)0;
                if (col + i < a.width) {
                    if (j == a.d) {
                        j = 0;
                        ++p;
                        k = equss::code_at(a.index, (int)p, r, a.K);
                    }
                    if (k != a.K) v[i] = from_f32<T>(to_f32<T>(books[((int64_t)p * a.K + k) * a.d + j]) * a.scale);
                    ++j;
                }
            }
            if (col + V <= a.width) {
                u32x4u2 w;
                if constexpr (T == 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, v[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        w[i] = (uint32_t)__builtin_bit_cast(u16, v[2 * i]) | (uint32_t)__builtin_bit_cast(u16, v[2 * i + 1]) << 16;
                }
                *reinterpret_cast<u32x4u2*>(dst) = w;
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (col + i < a.width) dst[i] = v[i];
            }
        }
    }
}

template <int T>
struct GradOp {
    const typename Elem<T>::type* g;
    int64_t ld;
    float scale;
    int d;
    typedef f32x4 Row;
    static constexpr bool kOwn = false;
    template <bool ONCE>
    __device__ __forceinline__ Row load(const equss::CodePair& at, int p, int col) const {
        const typename Elem<T>::type* s = g + (int64_t)at.row * ld + (int64_t)p * d + col;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (col + 4 <= d) {
            if constexpr (T == 0) {
                const f32x4u* from = reinterpret_cast<const f32x4u*>(s);
                const f32x4u w = ONCE ? __builtin_nontemporal_load(from) : *from;
                v = f32x4{w[0], w[1], w[2], w[3]};
            } else {
                const u32x2u2* from = reinterpret_cast<const u32x2u2*>(s);
                const u32x2u2 w = ONCE ? __builtin_nontemporal_load(from) : *from;
                if constexpr (T == 1) {
                    v = f32x4{equss::bits_as<float>(w[0] << 16), equss::bits_as<float>(w[0] & 0xffff0000u),
                              equss::bits_as<float>(w[1] << 16), equss::bits_as<float>(w[1] & 0xffff0000u)};
                } else {
                    const f16x2v lo = equss::bits_as<f16x2v>(w[0]), hi = equss::bits_as<f16x2v>(w[1]);
                    v = f32x4{(float)lo.x, (float)lo.y, (float)hi.x, (float)hi.y};
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + i < d) v[i] = to_f32<T>(s[i]);
        }
        return v;
    }
    __device__ __forceinline__ f32x4 value(Row& r) const { return r * scale; }
    template <bool ONCE>
    __device__ __forceinline__ void own(const Row&, uint32_t, int, int) const {}
};

int index_checks(const char* what, const void* idx, int index_type, int64_t rows, int num_pq, int64_t K, int d, int type) {
    if (rows < 0 || num_pq <= 0 || K <= 0 || d <= 0)
        return equss::fail(EQUSS_E_SHAPE, "%s: rows=%lld num_pq=%d K=%lld d=%d", what, (long long)rows, num_pq, (long long)K, d);
    if (index_type < EQUSS_I64 || index_type > EQUSS_I16 || type < EQUSS_F32 || type > EQUSS_F16)
        return equss::fail(EQUSS_E_UNSUPPORTED, "%s: index type %d, element type %d", what, index_type, type);
    if (num_pq > 65535 || d > (1 << 23) || (int64_t)num_pq * d > (1 << 24) || K >= ((int64_t)1 << 31) || rows > 0x7fffff00)
        return equss::fail(EQUSS_E_UNSUPPORTED, "%s: rows=%lld num_pq=%d K=%lld d=%d", what, (long long)rows, num_pq, (long long)K, d);
    if (rows > 0 && !idx) return equss::fail(EQUSS_E_NULL, "%s: null pointer argument", what);
    return EQUSS_OK;
}

template <int T>
int grad(const void* g, int64_t ld, float scale, const equss::SortPlan& s, const equss::IndexView& index, char* ws, float* out, int d, hipStream_t stream) {
    const GradOp<T> op = {reinterpret_cast<const typename Elem<T>::type*>(g), ld, scale, d};
    if (d <= 4) return equss::walk_launch_lpr<GradOp<T>, 1>(op, s, index, ws, out, d, stream);
    if (d <= 8) return equss::walk_launch_lpr<GradOp<T>, 2>(op, s, index, ws, out, d, stream);
    if (d <= 16) return equss::walk_launch_lpr<GradOp<T>, 4>(op, s, index, ws, out, d, stream);
    if (d <= 32) return equss::walk_launch_lpr<GradOp<T>, 8>(op, s, index, ws, out, d, stream);
    if (d <= 64) return equss::walk_launch_lpr<GradOp<T>, 16>(op, s, index, ws, out, d, stream);
    if (d <= 128) return equss::walk_launch_lpr<GradOp<T>, 32>(op, s, index, ws, out, d, stream);
    return equss::walk_launch_lpr<GradOp<T>, 64>(op, s, index, ws, out, d, stream);
}

}  // namespace

extern "C" int equss_code_lookup(const void* idx, int index_type, int64_t stride_p, int64_t stride_r, const void* books, int type,
                                 float scale, void* out, int64_t ld_out, int64_t rows, int num_pq, int64_t K, int d, void* stream) {
    const int rc = index_checks("equss_code_lookup", idx, index_type, rows, num_pq, K, d, type);
    if (rc != EQUSS_OK || rows == 0) return rc;
    if (!books || !out) return equss::fail(EQUSS_E_NULL, "equss_code_lookup: null pointer argument");
    const int es = type == EQUSS_F32 ? 4 : 2, v = 16 / es;
    LookupArgs a;
    a.index = {idx, index_type, stride_p, stride_r};
    a.books = books; a.out = out; a.ld_out = ld_out; a.rows = rows; a.scale = scale; a.num_pq = num_pq; a.d = d; a.K = (uint32_t)K;
    a.width = num_pq * d;
    if (ld_out < a.width || ((uintptr_t)books % 16) != 0 || ((uintptr_t)out % es) != 0)
        return equss::fail(EQUSS_E_ALIGN, "equss_code_lookup: books 16-byte aligned, rows of %d elements", a.width);
    a.units_row = (a.width + v - 1) / v;
    // (the division by units_code by multiplication: units_row * units_code below 2^32)
    const bool whole = (d % v) == 0 && (ld_out % v) == 0 && ((uintptr_t)out % 16) == 0 && (int64_t)a.units_row * (d / v) < ((int64_t)1 << 32);
    a.units_code = whole ? d / v : 1;
    int64_t r = 2048 / a.units_row;
    const int64_t spread = (rows + 2047) / 2048;
    if (r > spread) r = spread;
    if (r < 1) r = 1;
    // (the division by units_row: r * units_row <= 2048 units, or a row alone)
    a.rows_wg = (int)r;
    auto magic = [](int n) { return n == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + n - 1) / n); };
    a.magic_row = magic(a.units_row);
    a.magic_code = magic(a.units_code);
    if ((rows + r - 1) / r > equss::max_blocks(256))
        return equss::fail(EQUSS_E_UNSUPPORTED, "equss_code_lookup: %lld rows of %d elements", (long long)rows, a.width);
    const dim3 grid((unsigned)((rows + r - 1) / r));
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define EQUSS_LOOKUP(T)                                                                                 \
    if (whole) hipLaunchKernelGGL((code_lookup_kernel<T, true>), grid, dim3(256), 0, s, a);             \
    else hipLaunchKernelGGL((code_lookup_kernel<T, false>), grid, dim3(256), 0, s, a)
    if (type == EQUSS_F32) { EQUSS_LOOKUP(0); }
    else if (type == EQUSS_BF16) { EQUSS_LOOKUP(1); }
    else { EQUSS_LOOKUP(2); }
#undef EQUSS_LOOKUP
    return equss::check_launch("code_lookup_kernel");
}

extern "C" size_t equss_code_sums_sorted_workspace_bytes(int64_t rows, int num_pq, int64_t K, int d) {
    equss::SortPlan s;
    if (rows < 0 || num_pq <= 0 || K <= 0 || d <= 0 || !equss::sort_plan(s, rows, num_pq, K, d)) return 0;
    return s.total;
}

extern "C" int equss_code_lookup_grad(const void* g, int type, int64_t ld_g, const void* idx, int index_type, int64_t stride_p, int64_t stride_r,
                                      float scale, float* g_books, int64_t rows, int num_pq, int64_t K, int d, void* workspace,
                                      size_t workspace_bytes, void* stream) {
    const int rc = index_checks("equss_code_lookup_grad", idx, index_type, rows, num_pq, K, d, type);
    if (rc != EQUSS_OK) return rc;
    if (!g_books || (rows > 0 && !g)) return equss::fail(EQUSS_E_NULL, "equss_code_lookup_grad: null pointer argument");
    if (((uintptr_t)g_books % 16) != 0 || (rows > 0 && (ld_g < (int64_t)num_pq * d || ((uintptr_t)g % (type == EQUSS_F32 ? 4 : 2)) != 0)))
        return equss::fail(EQUSS_E_ALIGN, "equss_code_lookup_grad: g_books 16-byte aligned, rows of %lld elements", (long long)num_pq * d);
    equss::SortPlan s;
    if (!equss::sort_plan(s, rows, num_pq, K, d)) return equss::fail(EQUSS_E_UNSUPPORTED, "equss_code_lookup_grad: %lld rows", (long long)rows);
    if (s.total > 0 && (!workspace || workspace_bytes < s.total || ((uintptr_t)workspace % 256) != 0))
        return equss::fail(EQUSS_E_WORKSPACE, "equss_code_lookup_grad: workspace of %zu bytes, 256-byte aligned, needed", s.total);
    const equss::IndexView index = {idx, index_type, stride_p, stride_r};
    char* ws = reinterpret_cast<char*>(workspace);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (type == EQUSS_F32) return grad<0>(g, ld_g, scale, s, index, ws, g_books, d, st);
    if (type == EQUSS_BF16) return grad<1>(g, ld_g, scale, s, index, ws, g_books, d, st);
    return grad<2>(g, ld_g, scale, s, index, ws, g_books, d, st);
}
