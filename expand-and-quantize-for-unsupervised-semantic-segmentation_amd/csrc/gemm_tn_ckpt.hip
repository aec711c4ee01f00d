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
    int M, N, tiles_m, tiles_n, npad, mpad;
};

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

// C = sum of the partial products, in the order of the splits; then the bias
__global__ __launch_bounds__(256) void gemm_tn_join_kernel(const float* __restrict__ part, int64_t split_c, float* __restrict__ c,
                                                          int64_t ldc, const float* __restrict__ bpart, int64_t split_bias,
                                                          float* __restrict__ bias, int splits, int M, int N) {
    const int64_t cells = (int64_t)M * N;
    const int64_t total = cells + (bias ? M : 0);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const bool main = i < cells;
        const float* p = main ? part + i : bpart + (i - cells);
        const int64_t step = main ? split_c : split_bias;
        float s = 0.f;
        for (int k = 0; k < splits; ++k) s += p[k * step];
        if (main) c[(i / N) * ldc + i % N] = s;
        else bias[i - cells] = s;
    }
}

struct Plan { int tiles_m, tiles_n, splits; int64_t rows_split; };

Plan plan(int64_t rows, int M, int N) {
    Plan p;
    p.tiles_m = (M + TM - 1) / TM;
    p.tiles_n = (N + TN - 1) / TN;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    int64_t splits = (512 + tiles - 1) / tiles;
    const int64_t most = (rows + 4 * BK - 1) / (4 * BK);          // at least four steps a workgroup
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    p.rows_split = ((rows + splits - 1) / splits + BK - 1) / BK * BK;
    if (p.rows_split < BK) p.rows_split = BK;
    p.splits = (int)((rows + p.rows_split - 1) / p.rows_split);
    if (p.splits < 1) p.splits = 1;
    return p;
}

size_t workspace(const Plan& p, int M, int N) { return p.splits == 1 ? 0 : (size_t)p.splits * ((size_t)M * N + M) * sizeof(float); }

}  // namespace

extern "C" size_t equss_gemm_tn_ckpt_workspace_bytes(int64_t rows, int M, int N) {
    if (rows < 0 || M <= 0 || N <= 0) return 0;
    return workspace(plan(rows, M, N), M, N);
}

extern "C" int equss_gemm_tn_ckpt(const void* a, int64_t lda, const void* codes, int64_t ld_codes, const void* scales, int64_t ld_scales,
                                  int fmt, const void* relu_codes, int64_t ld_relu, float* C, int64_t ldc, float* bias, int64_t rows,
                                  int M, int N, void* workspace_ptr, size_t workspace_bytes, void* stream) {
    if (rows < 0 || M <= 0 || N <= 0) return equss::fail(EQUSS_E_SHAPE, "equss_gemm_tn_ckpt: rows=%lld M=%d N=%d", (long long)rows, M, N);
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
    const Plan p = plan(rows, M, N);
    const size_t need = workspace(p, M, N);
    if (need > 0 && (!workspace_ptr || workspace_bytes < need || ((uintptr_t)workspace_ptr % 16) != 0))
        return equss::fail(EQUSS_E_WORKSPACE, "equss_gemm_tn_ckpt: workspace of %zu bytes, 16-byte aligned, needed", need);
    const int64_t blocks = (int64_t)p.tiles_m * p.tiles_n * p.splits;
    if (blocks > 0x7fffffff || (p.rows_split + BK - 1) / BK > 0x7fffffff)
        return equss::fail(EQUSS_E_UNSUPPORTED, "equss_gemm_tn_ckpt: %lld rows, M=%d N=%d", (long long)rows, M, N);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    g.a = reinterpret_cast<const u16*>(a); g.lda = lda;
    g.codes = reinterpret_cast<const uint8_t*>(codes); g.ld_codes = ld_codes;
    g.scales = reinterpret_cast<const uint8_t*>(scales); g.ld_scales = ld_scales;
    g.mask = reinterpret_cast<const uint8_t*>(relu_codes); g.ld_mask = ld_relu;
    g.rows = rows; g.rows_split = p.rows_split; g.M = M; g.N = N; g.tiles_m = p.tiles_m; g.tiles_n = p.tiles_n;
    float* part = reinterpret_cast<float*>(workspace_ptr);
    float* bpart = part + (size_t)p.splits * M * N;
    const bool direct = p.splits == 1;
    g.c = direct ? C : part; g.ldc = direct ? ldc : N; g.split_c = direct ? 0 : (int64_t)M * N;
    g.bias = bias ? (direct ? bias : bpart) : nullptr; g.split_bias = direct ? 0 : M;
    const dim3 grid((unsigned)blocks), block(kTnThreads);
    if (fmt == EQUSS_CKPT_E4M3) {
        if (relu_codes) hipLaunchKernelGGL((gemm_tn_ckpt_kernel<true, true>), grid, block, 0, s, g);
        else hipLaunchKernelGGL((gemm_tn_ckpt_kernel<true, false>), grid, block, 0, s, g);
    } else {
        if (relu_codes) hipLaunchKernelGGL((gemm_tn_ckpt_kernel<false, true>), grid, block, 0, s, g);
        else hipLaunchKernelGGL((gemm_tn_ckpt_kernel<false, false>), grid, block, 0, s, g);
    }
    const int rc = equss::check_launch("gemm_tn_ckpt_kernel");
    if (rc != EQUSS_OK || direct) return rc;
    const int64_t total = (int64_t)M * N + (bias ? M : 0);
    int64_t gx = (total + 255) / 256;
    if (gx > 4096) gx = 4096;
    hipLaunchKernelGGL(gemm_tn_join_kernel, dim3((unsigned)gx), dim3(256), 0, s, part, (int64_t)M * N, C, ldc, bpart, (int64_t)M, bias,
                       p.splits, M, N);
    return equss::check_launch("gemm_tn_join_kernel");
}
