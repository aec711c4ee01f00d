// Backward of the training-pass quantisation (pq_backward.hip has the formulas) with the codes z kept in 8 bits, the codewords
// read from the codebooks instead of a saved copy, and the codebook gradient summed in a fixed order (code_sort.h).
//
// Rows are walked in the order of their codes, so a codeword is loaded once for a run of rows, the sum of (zn - emb) over the
// run stays in registers, and every (row, sub-space) is still visited once: its part of g_zq is read and its part of g_z
// written there.  A part is d consecutive elements (512 bytes of g_zq and g_z at d = 128): whole cache lines, so the order costs
// little extra traffic.  102400 rows, 8 x 256 x 128, int8: the walk takes 195 us with a gradient of z_q (955 MB at 4.9 TB/s; counted,
// 603 MB read and 427 written) and 102 without, as the training step has it; sort and join 24.  Bound by memory (a copy of 1 GiB:
// 5.15 TB/s).
//
// With n = max(|z|, 1e-12), zn = z / n, s = g_vq 2 / (rows d num_pq), the gradient of zn is g_zq + beta s (zn - emb), and
//     g_z = (g' - zn <zn, g'>) / n,   g' = g_zq - beta s emb
// since the projection removes what is parallel to zn: taken out before rather than cancelled after.  Where |z| < 1e-12 the
// norm is the constant 1e-12 (as F.normalize differentiates it): no projection.
#include "code_sort.h"

namespace {

struct PqArgs {
    const uint8_t* codes; int64_t ld_codes;
    const uint8_t* scales; int64_t ld_scales;
    const float* books;
    const float* g_zq; int64_t ld_g;
    const float* g_vq;
    float* g_z; int64_t ld_gz;
    float beta, book, inv_count;
    uint32_t K;
};

// HAS_G: a gradient arrives through the quantised output
template <bool E4M3, bool HAS_G, int D>
struct PqOp {
    PqArgs a;
    static constexpr int LPR = D / 4;
    static constexpr bool kOwn = true;
    // zn takes the place of the loads, g that of the output
    struct Row { uint32_t q, scale; f32x4 g, e; };
    template <bool ONCE>
    __device__ __forceinline__ Row load(const equss::CodePair& at, int p, int col) const {
        Row r;
        const int c = p * D + col;
        r.q = *reinterpret_cast<const uint32_t*>(a.codes + (int64_t)at.row * a.ld_codes + c);
        r.scale = a.scales[(int64_t)at.row * a.ld_scales + c / equss::kCkptBlock];
        r.g = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (HAS_G) {
            const f32x4* from = reinterpret_cast<const f32x4*>(a.g_zq + (int64_t)at.row * a.ld_g + c);
            r.g = ONCE ? __builtin_nontemporal_load(from) : *from;
        }
        r.e = f32x4{0.f, 0.f, 0.f, 0.f};
        if (at.code != a.K) r.e = *reinterpret_cast<const f32x4*>(a.books + ((int64_t)p * a.K + at.code) * D + col);
        return r;
    }
    __device__ __forceinline__ f32x4 value(Row& r) const {
        const float s = a.g_vq[0] * a.inv_count, bs = a.beta * s;
        const f32x4 z = equss::ckpt_decode4<E4M3>(r.q) * equss::ckpt_value_scale(r.scale);
        const float len = sqrtf(equss::lanes_sum<LPR>(z.x * z.x + z.y * z.y + z.z * z.z + z.w * z.w));
        const bool tiny = len < 1e-12f;
        const float inv = 1.f / (tiny ? 1e-12f : len);
        const f32x4 zn = z * inv;
        f32x4 g;
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = fmaf(-bs, r.e[i], r.g[i]);
        const float along = equss::lanes_sum<LPR>(zn.x * g.x + zn.y * g.y + zn.z * g.z + zn.w * g.w);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.g[i] = fmaf(zn[i], tiny ? bs : -along, g[i]) * inv;
        return (zn - r.e) * (-a.book * s);
    }
    template <bool ONCE>
    __device__ __forceinline__ void own(const Row& r, uint32_t row, int p, int col) const {
        if (!a.g_z) return;
        f32x4* to = reinterpret_cast<f32x4*>(a.g_z + (int64_t)row * a.ld_gz + p * D + col);
        if constexpr (ONCE) __builtin_nontemporal_store(r.g, to);
        else *to = r.g;
    }
};

template <int D>
int run(const PqArgs& a, bool e4m3, const equss::SortPlan& s, const equss::IndexView& index, char* ws, float* g_books, hipStream_t st) {
#define EQUSS_PQ(E, G) equss::walk_launch_lpr<PqOp<E, G, D>, D / 4>(PqOp<E, G, D>{a}, s, index, ws, g_books, D, st)
    if (e4m3) return a.g_zq ? EQUSS_PQ(true, true) : EQUSS_PQ(true, false);
    return a.g_zq ? EQUSS_PQ(false, true) : EQUSS_PQ(false, false);
#undef EQUSS_PQ
}

}  // namespace

extern "C" int equss_pq_st_backward_ckpt(const void* codes, int64_t ld_codes, const void* scales, int64_t ld_scales, int fmt,
                                         const float* books, const int64_t* idx, const float* g_zq, int64_t ld_g, const float* g_vq,
                                         float beta, float book, float* g_z, int64_t ld_gz, float* g_books, int64_t rows, int num_pq, int K,
                                         int d, void* workspace, size_t workspace_bytes, void* stream) {
    if (!codes || !scales || !books || !idx || !g_vq) return equss::fail(EQUSS_E_NULL, "equss_pq_st_backward_ckpt: null pointer argument");
    if (rows <= 0 || num_pq <= 0 || K <= 0)
        return equss::fail(EQUSS_E_SHAPE, "equss_pq_st_backward_ckpt: rows=%lld num_pq=%d K=%d", (long long)rows, num_pq, K);
    if (d != 16 && d != 32 && d != 64 && d != 128)
        return equss::fail(EQUSS_E_UNSUPPORTED, "equss_pq_st_backward_ckpt: sub-space dim %d (16, 32, 64 or 128)", d);
    if (fmt != EQUSS_CKPT_INT8 && fmt != EQUSS_CKPT_E4M3) return equss::fail(EQUSS_E_UNSUPPORTED, "equss_pq_st_backward_ckpt: format %d", fmt);
    const int64_t cols = (int64_t)num_pq * d, padded = (cols + equss::kCkptBlock - 1) / equss::kCkptBlock * equss::kCkptBlock;
    equss::SortPlan s;
    if (cols > (1 << 24) || !equss::sort_plan(s, rows, num_pq, K, d))
        return equss::fail(EQUSS_E_UNSUPPORTED, "equss_pq_st_backward_ckpt: rows=%lld num_pq=%d", (long long)rows, num_pq);
    auto bad = [&](const float* p, int64_t ld) { return p && (ld < cols || (ld % 4) != 0 || ((uintptr_t)p % 16) != 0); };
    if (bad(g_zq, ld_g) || bad(g_z, ld_gz) || ld_codes < padded || (ld_codes % equss::kCkptBlock) != 0 || ((uintptr_t)codes % 16) != 0 ||
        ld_scales < padded / equss::kCkptBlock || ((uintptr_t)books % 16) != 0 || ((uintptr_t)g_books % 16) != 0)
        return equss::fail(EQUSS_E_ALIGN, "equss_pq_st_backward_ckpt: buffers 16-byte aligned, leading dimensions of rows >= num_pq * d and multiples "
                           "of 4, of codes >= %lld and multiples of 32", (long long)padded);
    if (s.total > 0 && (!workspace || workspace_bytes < s.total || ((uintptr_t)workspace % 256) != 0))
        return equss::fail(EQUSS_E_WORKSPACE, "equss_pq_st_backward_ckpt: workspace of %zu bytes, 256-byte aligned, needed", s.total);
    if (!g_z && !g_books) return EQUSS_OK;
    PqArgs a;
    a.codes = reinterpret_cast<const uint8_t*>(codes); a.ld_codes = ld_codes;
    a.scales = reinterpret_cast<const uint8_t*>(scales); a.ld_scales = ld_scales;
    a.books = books; a.g_zq = g_zq; a.ld_g = ld_g; a.g_vq = g_vq; a.g_z = g_z; a.ld_gz = ld_gz;
    a.beta = beta; a.book = book; a.inv_count = (float)(2.0 / ((double)rows * d * num_pq)); a.K = (uint32_t)K;
    const equss::IndexView index = {idx, EQUSS_I64, rows, 1};
    char* ws = reinterpret_cast<char*>(workspace);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const bool e = fmt == EQUSS_CKPT_E4M3;
    switch (d) {
        case 16: return run<16>(a, e, s, index, ws, g_books, st);
        case 32: return run<32>(a, e, s, index, ws, g_books, st);
        case 64: return run<64>(a, e, s, index, ws, g_books, st);
        default: return run<128>(a, e, s, index, ws, g_books, st);
    }
}
