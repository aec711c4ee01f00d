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
    int M, N, tiles_m, tiles_n, splits, npad, mpad;
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

// ---- the large tile: 4 waves of WM x WN MFMA tiles of 32 x 32, i.e. 64 WM x 64 WN of C; 32 rows a stage, three stages in LDS.
// A wave's accumulators take up to 256 registers, so there is one wave a SIMD, and what hides its latencies is its own pipeline.
// While a stage's fragments are multiplied,
//   the fragments of the next half stage are read (the next stage's first half too: its writes are a barrier back),
//   the stage after the next goes from registers through the conversion into the third slot of LDS, and
//   each of those registers is requested again from two stages further on (there are two sets of them: one stage of 32 rows
//   takes half a microsecond, less than a load from memory does under load),
// without a branch in between, so that the scheduler can put all of it between the MFMAs.
// Columns past M: the last chunk of 8 columns is read at M - 8, so that every load is whole and inside; its columns then
// overlap the chunk before, both give the same sums, and both are written.  Columns past N lie in the checkpoint's padding or
// are read from its last block; their sums are dropped.
constexpr int kBigBK = 32, kSlots = 3;

template <int T64> struct TileRow { static constexpr int bytes = T64 == 2 ? 256 : 512; };   // (192 columns in rows of 512: the swizzle's xor needs them)

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

template <bool E4M3, bool MASK, int WM, int WN>
__global__ __launch_bounds__(256, 1) void gemm_tn_ckpt_big_kernel(const Args g) {
    constexpr int TMB = 64 * WM, TNB = 64 * WN, RA = TileRow<WM>::bytes, RB = TileRow<WN>::bytes;
    constexpr int SLOT = kBigBK * (RA + RB);
    constexpr int ACH = RA / 16, BCH = RB / 32;             // a row's chunks of 8 columns of a, of 16 codes
    constexpr int AP = kBigBK * ACH / 256, BP = kBigBK * BCH / 256;   // passes of the 256 threads over a stage
    constexpr int AROWS = 256 / ACH, BROWS = 256 / BCH;     // rows a pass
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
    const int rows = (int)(k1 - k0);
    const int stages = (rows + kBigBK - 1) / kBigBK, whole = rows / kBigBK;

    // ---- staging.  Addresses are a uniform part (stage and pass) and a lane's 32-bit offset within a stage.
    const int ach = tid % ACH, arow = tid / ACH, bch = tid % BCH, brow = tid / BCH;
    int ma = m0 + 8 * ach, nb = n0 + 16 * bch;
    ma = ma + 8 <= g.M ? ma : g.M - 8;
    nb = nb + 16 <= g.npad ? nb : g.npad - 16;
    const int lda = (int)g.lda, ldc = (int)g.ld_codes, lds = (int)g.ld_scales, ldm = (int)g.ld_mask;
    const uint32_t va = (uint32_t)((arow * lda + ma) * 2), vm = (uint32_t)(arow * ldm + ma);
    const uint32_t vb = (uint32_t)(brow * ldc + nb), vs = (uint32_t)(brow * lds + nb / equss::kCkptBlock);
    u32x4a ra[2][AP], rb[2][BP];
    uint2 rm[2][AP];
    uint32_t rs[2][BP];
    typedef uint32_t u32x2u1 __attribute__((ext_vector_type(2), aligned(1)));
    // LAST: the stage's rows may end before its 32: the others repeat the last one (and are zeroed on their way into LDS)
    auto load_a = [&](auto last_c, int set, int i, int stage) __attribute__((always_inline)) {
        constexpr bool LAST = decltype(last_c)::value;
        const int64_t row = k0 + (int64_t)stage * kBigBK + (LAST ? 0 : AROWS * i);
        uint32_t oa = va, om = vm;
        if constexpr (LAST) {
            const int left = rows - stage * kBigBK - 1, r = arow + AROWS * i < left ? arow + AROWS * i : left;
            oa = (uint32_t)((r * lda + ma) * 2);
            om = (uint32_t)(r * ldm + ma);
        }
        const u32x4u2 v = *reinterpret_cast<const u32x4u2*>(reinterpret_cast<const char*>(g.a + row * g.lda) + oa);
        ra[set][i] = u32x4a{v[0], v[1], v[2], v[3]};
        if constexpr (MASK) {
            const u32x2u1 c = *reinterpret_cast<const u32x2u1*>(g.mask + row * g.ld_mask + om);
            rm[set][i] = make_uint2(c[0], c[1]);
        }
    };
    auto load_b = [&](auto last_c, int set, int i, int stage) __attribute__((always_inline)) {
        constexpr bool LAST = decltype(last_c)::value;
        const int64_t row = k0 + (int64_t)stage * kBigBK + (LAST ? 0 : BROWS * i);
        uint32_t ob = vb, os = vs;
        if constexpr (LAST) {
            const int left = rows - stage * kBigBK - 1, r = brow + BROWS * i < left ? brow + BROWS * i : left;
            ob = (uint32_t)(r * ldc + nb);
            os = (uint32_t)(r * lds + nb / equss::kCkptBlock);
        }
        rb[set][i] = *reinterpret_cast<const u32x4a*>(g.codes + row * g.ld_codes + ob);
        rs[set][i] = (g.scales + row * g.ld_scales)[os];
    };
    float bsum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) bsum[j] = 0.f;
    // the bias: every tile of a row of tiles adds up its share of the stages, [bias0, bias1); even ones, as the loop goes by two
    const int bias0 = g.bias ? (int)((int64_t)stages * tn / g.tiles_n) & ~1 : 0;
    const int bias1 = !g.bias ? 0 : tn + 1 == g.tiles_n ? stages : (int)((int64_t)stages * (tn + 1) / g.tiles_n) & ~1;
    auto store_a = [&](auto last_c, auto bias_c, int set, int i, int stage, char* sb) __attribute__((always_inline)) {
        const int r = arow + AROWS * i;
        u32x4a v = ra[set][i];
        if constexpr (MASK) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w = (j & 2 ? rm[set][i].y : rm[set][i].x) >> (16 * (j & 1));
                v[j] &= ((int8_t)w > 0 ? 0xffffu : 0u) | ((int8_t)(w >> 8) > 0 ? 0xffff0000u : 0u);
            }
        }
        if constexpr (decltype(last_c)::value) {
            if (stage * kBigBK + r >= rows) v = u32x4a{0, 0, 0, 0};
        }
        if constexpr (decltype(bias_c)::value) {
            const uint32_t mine = !decltype(last_c)::value || (stage >= bias0 && stage < bias1) ? 0xffffffffu : 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                bsum[2 * j] += equss::bits_as<float>((v[j] & mine) << 16);
                bsum[2 * j + 1] += equss::bits_as<float>(v[j] & mine & 0xffff0000u);
            }
        }
        *reinterpret_cast<u32x4a*>(sb + r * RA + ((ach ^ (4 * (r & 3))) * 16)) = v;
    };
    auto store_b = [&](auto last_c, int set, int i, int stage, char* sb) __attribute__((always_inline)) {
        const int r = brow + BROWS * i;
        uint32_t sc = rs[set][i];
        u32x4a c = rb[set][i];
        if constexpr (decltype(last_c)::value) {
            if (stage * kBigBK + r >= rows) { sc = 0; c = u32x4a{0, 0, 0, 0}; }
        }
        const float s = equss::ckpt_scale(sc);
        char* row = sb + kBigBK * RA + r * RB;
        *reinterpret_cast<u32x4a*>(row + (((2 * bch) ^ (4 * (r & 3))) * 16)) = to_bf16x8<E4M3>(c[0], c[1], s);
        *reinterpret_cast<u32x4a*>(row + (((2 * bch + 1) ^ (4 * (r & 3))) * 16)) = to_bf16x8<E4M3>(c[2], c[3], s);
    };

    const int wm = wave >> 1, wn = wave & 1;
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
    int a_at[WM], b_at[WN];
#pragma unroll
    for (int t = 0; t < WM; ++t) a_at[t] = frag_at((wm * WM + t) * 32, RA);
#pragma unroll
    for (int t = 0; t < WN; ++t) b_at[t] = kBigBK * RA + frag_at((wn * WN + t) * 32, RB);
    bf16x8 af[2][WM], bf[2][WN];
    auto read = [&](int set, const char* slot, int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < WM; ++t) af[set][t] = frag(slot + ks * 16 * RA + a_at[t], RA);
#pragma unroll
        for (int t = 0; t < WN; ++t) bf[set][t] = frag(slot + ks * 16 * RB + b_at[t], RB);
    };
    f32x16 acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    auto multiply = [&](int set) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < WM; ++i)
#pragma unroll
            for (int j = 0; j < WN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[set][i], bf[set][j], acc[i][j], 0, 0, 0);
    };
    using No = std::false_type;
    using Yes = std::true_type;
    auto fetch = [&](int set, int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AP; ++i) load_a(Yes(), set, i, stage);
#pragma unroll
        for (int i = 0; i < BP; ++i) load_b(Yes(), set, i, stage);
    };
    auto put = [&](int set, int stage, char* slot) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AP; ++i) store_a(Yes(), Yes(), set, i, stage, slot);
#pragma unroll
        for (int i = 0; i < BP; ++i) store_b(Yes(), set, i, stage, slot);
    };
    // one stage: multiply `stage`, read ahead, store stage + 2 and request stage + 4 (which are there and whole)
    auto step = [&](auto bias_c, int set, int stage, const char* s0, const char* s1, char* s2) __attribute__((always_inline)) {
        const No last_c;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (ks == 0) read(1, s0, 1);
            else read(0, s1, 0);
#pragma unroll
            for (int i = ks * AP / 2; i < (ks + 1) * AP / 2; ++i) { store_a(last_c, bias_c, set, i, stage + 2, s2); load_a(last_c, set, i, stage + 4); }
#pragma unroll
            for (int i = ks * BP / 2; i < (ks + 1) * BP / 2; ++i) { store_b(last_c, set, i, stage + 2, s2); load_b(last_c, set, i, stage + 4); }
            multiply(ks);
            // the order wanted: behind every MFMA two fragment reads (first half) or a store and its next request, and conversions
#pragma unroll
            for (int i = 0; i < WM * WN; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);            // MFMA
                if (i < WM + WN) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // LDS reads
                __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);            // VALU
                if (i >= WM * WN / 2) {
                    __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);        // LDS write
                    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);        // global load
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
    };

    if (stages > 0) {
        fetch(0, 0);
        if (stages > 1) fetch(1, 1);
        put(0, 0, smem);
        if (stages > 2) fetch(0, 2);
        if (stages > 1) put(1, 1, smem + SLOT);
        if (stages > 3) fetch(1, 3);
    }
    __syncthreads();
    if (stages > 0) read(0, smem, 0);
    int stage = 0, slot = 0;
    auto at = [&](int k) __attribute__((always_inline)) { return smem + (slot + k >= kSlots ? slot + k - kSlots : slot + k) * SLOT; };
    auto next = [&]() __attribute__((always_inline)) {
        ++stage;
        slot = slot + 1 == kSlots ? 0 : slot + 1;
    };
    const int end = whole - 4;
    auto run = [&](auto bias_c, int to) __attribute__((always_inline)) {
        while (stage + 1 < to) {
            step(bias_c, 0, stage, at(0), at(1), at(2));
            next();
            step(bias_c, 1, stage, at(0), at(1), at(2));
            next();
        }
    };
    run(No(), end < bias0 - 2 ? end : bias0 - 2);
    run(Yes(), end < bias1 - 2 ? end : bias1 - 2);
    run(No(), end);
    auto last = [&](int set) __attribute__((always_inline)) {                              // the last few, one thing after the other
        if (stage + 2 < stages) put(set, stage + 2, at(2));
        if (stage + 4 < stages) fetch(set, stage + 4);
        read(1, at(0), 1);
        multiply(0);
        if (stage + 1 < stages) read(0, at(1), 0);
        multiply(1);
        __syncthreads();
        next();
    };
    while (stage < stages) {
        last(0);
        if (stage < stages) last(1);
    }

    float* c = g.c + split * g.split_c;
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int chunk = m0 + (wm * WM + i) * 32 + 8 * (r >> 2);
            if (chunk < g.M) {
                const int m = (chunk + 8 <= g.M ? chunk : g.M - 8) + 4 * kb + (r & 3);
#pragma unroll
                for (int j = 0; j < WN; ++j) {
                    const int n = n0 + (wn * WN + j) * 32 + (lane & 31);
                    if (n < g.N) c[m * g.ldc + n] = acc[i][j][r];
                }
            }
        }
    if (g.bias) {
        float* part = reinterpret_cast<float*>(smem);      // (every reader of the tiles is behind the loop's last barrier)
#pragma unroll
        for (int j = 0; j < 8; ++j) part[arow * (8 * ACH) + 8 * ach + j] = bsum[j];
        __syncthreads();
        const int chunk = m0 + tid / 8 * 8;
        if (tid < TMB && chunk < g.M) {
            float s = 0.f;
            for (int r = 0; r < AROWS; ++r) s += part[r * (8 * ACH) + tid];
            g.bias[(split * g.tiles_n + tn) * g.split_bias + (chunk + 8 <= g.M ? chunk : g.M - 8) + tid % 8] = s;
        }
    }
}

// C = sum of the partial products, in the order of the splits; then the bias
__global__ __launch_bounds__(256) void gemm_tn_join_kernel(const float* __restrict__ part, int64_t split_c, float* __restrict__ c,
                                                          int64_t ldc, const float* __restrict__ bpart, int64_t split_bias,
                                                          float* __restrict__ bias, int splits, int bias_splits, int M, int N, int bias_len) {
    const int64_t cells = (int64_t)M * N;
    const int64_t total = cells + (bias ? bias_len : 0);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const bool main = i < cells;
        const float* p = main ? part + i : bpart + (i - cells);
        const int64_t step = main ? split_c : split_bias;
        const int n = main ? splits : bias_splits;
        float s = 0.f;
        int k = 0;
        for (; k + 8 <= n; k += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = p[(k + j) * step];
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[j];
        }
        for (; k < n; ++k) s += p[k * step];
        if (main) c[(i / N) * ldc + i % N] = s;
        else bias[i - cells] = s;
    }
}

struct Plan { bool big; int tiles_m, tiles_n, splits, bias_splits; int64_t rows_split; };

Plan plan(int64_t rows, int M, int N) {
    Plan p;
    p.big = M > 128 && N > 128;
    const int tm = p.big ? 256 : TM, tn = p.big ? 256 : TN, bk = p.big ? kBigBK : BK;
    p.tiles_m = (M + tm - 1) / tm;
    p.tiles_n = (N + tn - 1) / tn;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    int64_t splits = p.big ? 256 / tiles : (512 + tiles - 1) / tiles;
    const int64_t most = (rows + 4 * bk - 1) / (4 * bk);          // at least four steps a workgroup
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    p.rows_split = ((rows + splits - 1) / splits + bk - 1) / bk * bk;
    if (p.rows_split < bk) p.rows_split = bk;
    p.splits = (int)((rows + p.rows_split - 1) / p.rows_split);
    if (p.splits < 1) p.splits = 1;
    p.bias_splits = p.big ? p.splits * p.tiles_n : p.splits;
    return p;
}

// partial products and, behind them, partial bias sums; nothing where one row range and one tile across write the results
size_t workspace(const Plan& p, int M, int N) {
    const size_t c = p.splits == 1 ? 0 : (size_t)p.splits * M * N, b = p.bias_splits == 1 ? 0 : (size_t)p.bias_splits * M;
    return (c + b) * sizeof(float);
}

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
    // (offsets within a stage of 64 rows are 32 bits)
    if (rows > 0 && (lda > (1 << 23) || ld_codes > (1 << 23) || ld_relu > (1 << 23)))
        return equss::fail(EQUSS_E_UNSUPPORTED, "equss_gemm_tn_ckpt: a leading dimension exceeds %d", 1 << 23);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    g.a = reinterpret_cast<const u16*>(a); g.lda = lda;
    g.codes = reinterpret_cast<const uint8_t*>(codes); g.ld_codes = ld_codes;
    g.scales = reinterpret_cast<const uint8_t*>(scales); g.ld_scales = ld_scales;
    g.mask = reinterpret_cast<const uint8_t*>(relu_codes); g.ld_mask = ld_relu;
    g.rows = rows; g.rows_split = p.rows_split; g.M = M; g.N = N; g.tiles_m = p.tiles_m; g.tiles_n = p.tiles_n; g.splits = p.splits;
    float* part = reinterpret_cast<float*>(workspace_ptr);
    float* bpart = part + (p.splits == 1 ? 0 : (size_t)p.splits * M * N);
    const bool direct = p.splits == 1, bias_direct = p.bias_splits == 1;
    g.c = direct ? C : part; g.ldc = direct ? ldc : N; g.split_c = direct ? 0 : (int64_t)M * N;
    g.bias = bias ? (bias_direct ? bias : bpart) : nullptr; g.split_bias = M;
    const bool e = fmt == EQUSS_CKPT_E4M3;
    if (p.big) {
        const int lds = kSlots * kBigBK * 1024;
        const dim3 grid((unsigned)((blocks + 7) / 8 * 8));
#define EQUSS_TN_BIG(E, K)                                                                                                     \
    do {                                                                                                                       \
        if (!equss::lds_opt_in(reinterpret_cast<const void*>(&gemm_tn_ckpt_big_kernel<E, K, 4, 4>), lds))                      \
            return equss::fail(EQUSS_E_UNSUPPORTED, "equss_gemm_tn_ckpt: %d bytes of LDS", lds);                               \
        hipLaunchKernelGGL((gemm_tn_ckpt_big_kernel<E, K, 4, 4>), grid, dim3(256), lds, s, g);                                 \
    } while (0)
        if (e) { if (relu_codes) EQUSS_TN_BIG(true, true); else EQUSS_TN_BIG(true, false); }
        else { if (relu_codes) EQUSS_TN_BIG(false, true); else EQUSS_TN_BIG(false, false); }
#undef EQUSS_TN_BIG
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
    const bool join_bias = bias && !bias_direct;
    if (rc != EQUSS_OK || (direct && !join_bias)) return rc;
    // (with one row range the products are in place and only the bias is left)
    const int64_t total = (direct ? 0 : (int64_t)M * N) + (join_bias ? M : 0);
    int64_t gx = (total + 255) / 256;
    if (gx > 4096) gx = 4096;
    hipLaunchKernelGGL(gemm_tn_join_kernel, dim3((unsigned)gx), dim3(256), 0, s, part, (int64_t)M * N, C, ldc, bpart, (int64_t)M,
                       join_bias ? bias : nullptr, p.splits, p.bias_splits, direct ? 0 : M, direct ? 1 : N, M);
    return equss::check_launch("gemm_tn_join_kernel");
}
