// Sums over the rows of every code, in a fixed order: what the gradient of a codeword lookup is, and the codebook gradient of
// the quantiser's backward.  Float atomics would do it in one pass, but in the order of their arrival, and the codes of a
// batch are used unevenly, so that the busiest codeword's adders queue.  Instead the rows are put in the order of their codes
// (a stable radix sort of (code, row) pairs, 8 bytes each against the hundreds of bytes of a row) and walked in that order:
//
//   count      a histogram of the digit for every chunk of rows
//   place      every chunk's pairs to their place: bin start + the bin's pairs of earlier chunks + rank within the chunk
//              (two passes of up to 11 bits for more than 2047 codes, three beyond 4 million; one kernel that finds the runs)
//   accumulate tiles of T sorted pairs, T the same for every tile however the codes are used; a group of lanes walks one tile and
//              keeps the running sum in registers.  A code's run that lies within a tile is written at once; one that crosses
//              tile borders leaves a partial sum on each
//   join       the partial sums of a run in the order of the tiles, and zeros for codes without rows
//
// For few rows all of it is one kernel (small): a workgroup owns a few codes, picks their rows out of all indices by itself, in
// order, and sums them.  Measured (us a call, small against sorted; codes used evenly, by the square of a uniform number, all rows of
// one code), gradient of a lookup, 8 x 256 x 128: 1024 rows 8.9 / 18, 13 / 18, 32 / 20; 2048 rows 9.8 / 19, 16 / 19, 54 / 21; 4096
// rows, even and one code: 22 / 22, 92 / 29; quantiser's backward: 1024 rows 13 / 23, 19 / 23, 107 / 23; 2048 rows 13 / 23, 28 / 23,
// 207 / 25.  4096 rows, 16384 x 16, whose sort takes two passes: 12 / 38.  Hence up to 2048 rows, and up to 4096 where the sort
// would take more than one pass.  What it costs at worst goes by the rows of the busiest workgroup, not by the codes: 4096 rows on
// 150000 x 32, even use, 300 neighbouring codes, one code: 17, 37, 37; on 5 million x 8: 51, 105, 90.
//
// An index outside [0, K) counts as the code K, which sorts last and has no sum.
#pragma once
#include "ckpt.h"

namespace equss {

struct IndexView {            // (num_pq, rows) indices of any integer type and any strides (in elements)
    const void* p;
    int type;                 // EQUSS_I64 / EQUSS_I32 / EQUSS_I16
    int64_t stride_p, stride_r;
};

__device__ __forceinline__ uint32_t code_at(const IndexView& v, int p, int64_t r, uint32_t K) {
    const int64_t at = (int64_t)p * v.stride_p + r * v.stride_r;
    int64_t k;
    if (v.type == EQUSS_I64) k = reinterpret_cast<const int64_t*>(v.p)[at];
    else if (v.type == EQUSS_I32) k = reinterpret_cast<const int32_t*>(v.p)[at];
    else k = reinterpret_cast<const int16_t*>(v.p)[at];
    return k >= 0 && k < (int64_t)K ? (uint32_t)k : K;
}

// The codes of rows r, r + step, ... (N of them; those past `end` give the last row's): the loads of one type side by side, so
// that they wait once, not N times.
template <int N>
__device__ __forceinline__ void codes_at(const IndexView& v, int p, int64_t r, int step, int64_t end, uint32_t K, uint32_t (&code)[N]) {
    int64_t k[N];
    auto load = [&](auto* base) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int64_t at = r + (int64_t)j * step < end ? r + (int64_t)j * step : end - 1;
            k[j] = base[at * v.stride_r];
        }
    };
    const int64_t first = (int64_t)p * v.stride_p;
    if (v.type == EQUSS_I64) load(reinterpret_cast<const int64_t*>(v.p) + first);
    else if (v.type == EQUSS_I32) load(reinterpret_cast<const int32_t*>(v.p) + first);
    else load(reinterpret_cast<const int16_t*>(v.p) + first);
#pragma unroll
    for (int j = 0; j < N; ++j) code[j] = k[j] >= 0 && k[j] < (int64_t)K ? (uint32_t)k[j] : K;
}

struct CodePair { uint32_t code, row; };

constexpr int kSmallRows = 4096;        // most rows of the one-kernel form
constexpr int kMaxBins = 2048;          // bins of a pass: 11 bits
constexpr int kTile = 64;               // pairs of a tile, where there are enough of them

// What a call sorts with; everything but `index` lies in the caller's workspace.
struct SortPlan {
    int64_t rows;
    int num_pq;
    uint32_t K;
    int passes, bits[3];
    int chunks, chunk_rows;             // chunk_rows a multiple of 256
    int tile;                           // T
    int64_t tiles;
    size_t pairs_a, pairs_b, table, starts, partial, total;   // byte offsets and the whole size
};

// d: elements of a row's part.  False where sizes pass what the kernels index with.
bool sort_plan(SortPlan& s, int64_t rows, int num_pq, int64_t K, int d);
// count / place (/ runs): afterwards the sorted pairs are at ws + the returned offset and starts at ws + s.starts
int sort_launch(const SortPlan& s, const IndexView& index, char* ws, size_t* pairs_at, hipStream_t stream);

// --------------------------------------------------------------------------------------------------------------------------
// The walk.  Op gives the kernels their rows:
//   struct Row;                             what is loaded of one (code, row) pair and lane
//   Row  load<ONCE>(pair, p, col) const     its loads; ONCE: more data than the caches hold, past them where a row is not shared
//   f32x4 value(const Row&) const           the lane's four terms of the sum
//   kOwn; own<ONCE>(const Row&, row, p, col)   whether a row has an output of its own, and its store; after value(), which may
//                                           leave what it needs in Row
// A row's part of d elements is walked by LPR lanes with four elements each (d <= 4 LPR; beyond 256 in chunks of 256 columns).

struct WalkArgs {
    const CodePair* pairs;              // (num_pq, rows)
    const uint32_t* starts;             // (num_pq, K + 1)
    float* partial;                     // (num_pq, tiles, 2, dpad): a tile's head and tail
    float* out;                         // (num_pq, K, d), or null: only the rows' own outputs are wanted
    int64_t rows, tiles;
    int64_t code0;                      // the join's first code
    int tile, d, dpad;
    uint32_t K;
};

__device__ __forceinline__ void store_cols(float* p, f32x4 v, int col, int d, bool whole) {
    if (whole) *reinterpret_cast<f32x4*>(p) = v;          // (d a multiple of 4: 16-byte aligned)
    else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col + i < d) p[i] = v[i];
    }
}

// U: pairs in flight a group.  One where the chip is full of groups (102400 rows, 8 x 256 x 128, the quantiser's backward: 223 us
// with 1, 251 with 2, 267 with 4), two where it is not (4096 rows: 33 / 30 / 31 us).  The rows of the first kind go past the
// caches (lookup gradient of 102400 rows: 99 us, 110 us through them; of 16384 rows: 33 / 32 us).
template <class Op, int LPR, int U>
__global__ __launch_bounds__(256) void code_accumulate_kernel(const Op op, const WalkArgs w) {
    constexpr int SLOTS = 64 / LPR;
    const int lane = threadIdx.x & 63;
    const int64_t tile = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * SLOTS + lane / LPR;
    if (tile >= w.tiles) return;                          // (whole groups of LPR lanes leave together)
    const int p = blockIdx.y, col = (int)blockIdx.z * 256 + (lane % LPR) * 4;
    const bool live = col < w.d, whole = (w.d & 3) == 0;
    const CodePair* pairs = w.pairs + (int64_t)p * w.rows;
    const int64_t t0 = tile * w.tile, t1 = t0 + w.tile < w.rows ? t0 + w.tile : w.rows;
    uint32_t cur = pairs[t0].code;
    bool head = t0 > 0 && pairs[t0 - 1].code == cur;      // the run began in an earlier tile
    float* part = w.partial + (((int64_t)p * w.tiles + tile) * 2) * w.dpad + col;
    float* out = w.out + ((int64_t)p * w.K) * w.d + col;
    const bool sums = w.out != nullptr;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    CodePair next[U];
#pragma unroll
    for (int j = 0; j < U; ++j) next[j] = pairs[t0 + j < t1 ? t0 + j : t1 - 1];
    for (int64_t i = t0; i < t1; i += U) {
        CodePair pr[U];
        typename Op::Row row[U];
        f32x4 v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            pr[j] = next[j];
            row[j] = op.template load<U == 1>(pr[j], p, live ? col : 0);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) next[j] = pairs[i + U + j < t1 ? i + U + j : t1 - 1];
        // (a pair past the tile's end is its last one again: its value is not used and its own output is the same once more)
#pragma unroll
        for (int j = 0; j < U; ++j) v[j] = op.value(row[j]);
#pragma unroll
        for (int j = 0; j < U; ++j) op.template own<U == 1>(row[j], pr[j].row, p, col);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (i + j < t1) {
                if (pr[j].code != cur) {
                    if (sums && live && cur != w.K) {
                        if (head) *reinterpret_cast<f32x4*>(part) = acc;
                        else store_cols(out + (int64_t)cur * w.d, acc, col, w.d, whole);
                    }
                    head = false;
                    cur = pr[j].code;
                    acc = f32x4{0.f, 0.f, 0.f, 0.f};
                }
                acc += v[j];
            }
        }
    }
    if (sums && live && cur != w.K) {
        const bool on = t1 < w.rows && pairs[t1].code == cur;
        if (head) *reinterpret_cast<f32x4*>(part) = acc;
        else if (on) *reinterpret_cast<f32x4*>(part + w.dpad) = acc;
        else store_cols(out + (int64_t)cur * w.d, acc, col, w.d, whole);
    }
}

// WAVES = 4: a wave owns a code, and the chain of partial sums of a long run is shared by the workgroup's four waves.  WAVES = 16,
// where there are few codes, i.e. long runs: a workgroup owns a code (102045 rows, 5 x 2 x 32, gradient of a lookup: 42 us, 65 us
// with four waves; 102400 rows, 8 x 256 x 128: 100 / 96 us, hence at most 1024 codes), and at most 2048 workgroups, a codeword of
// more than 256 columns taking several (3000 rows, 1000 x 4096, 16000 workgroups: 81 us, 36 with four waves each; 20000 rows of one
// code, 600 x 512, 1200 workgroups: 55 / 74).
template <int LPR, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void code_join_kernel(const WalkArgs w) {
    constexpr int SLOTS = 64 / LPR, CODES = WAVES == 4 ? 4 : 1, kLong = 16 * SLOTS, F = 8;
    __shared__ f32x4 share[WAVES][LPR];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slot = lane / LPR;
    const int p = blockIdx.y, col = (int)blockIdx.z * 256 + (lane % LPR) * 4;
    const bool live = col < w.d, whole = (w.d & 3) == 0;
    const uint32_t* starts = w.starts + (int64_t)p * ((int64_t)w.K + 1);
    const float* part = w.partial + (int64_t)p * w.tiles * 2 * w.dpad + (live ? col : 0);
    float* out = w.out + (int64_t)p * w.K * w.d + col;
    // link 0 is the first tile's tail, the others the following tiles' heads; the sum of links first, first + step, ... of all the
    // groups of a wave, in every one of them
    auto chain = [&](int64_t ts, int64_t links, int64_t first, int64_t step) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int64_t j = first; j < links; j += F * step) {
            f32x4 v[F];
#pragma unroll
            for (int i = 0; i < F; ++i) {
                const int64_t l = j + i * step < links ? j + i * step : first;
                v[i] = *reinterpret_cast<const f32x4*>(part + ((ts + l) * 2 + (l == 0 ? 1 : 0)) * w.dpad);
            }
#pragma unroll
            for (int i = 0; i < F; ++i)
                if (j + i * step < links) acc += v[i];
        }
#pragma unroll
        for (int o = 32; o >= LPR; o >>= 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], o, 64);
        return acc;
    };
    const int64_t k0 = w.code0 + (int64_t)blockIdx.x * CODES;
    int64_t at[CODES + 1];
#pragma unroll
    for (int c = 0; c <= CODES; ++c) at[c] = starts[k0 + c <= (int64_t)w.K ? k0 + c : (int64_t)w.K];
#pragma unroll
    for (int c = 0; c < CODES; ++c) {
        const int64_t k = k0 + c;
        if (k >= (int64_t)w.K) break;                      // (uniform over the workgroup)
        const int64_t s = at[c], e = at[c + 1];
        const int64_t ts = s / w.tile, links = e > s ? (e - 1) / w.tile - ts + 1 : 0;
        if (links <= kLong) {
            if (wave != c || links == 1) continue;         // one tile held the whole run: it is written already
            const f32x4 acc = chain(ts, links, slot, SLOTS);
            if (slot == 0 && live) store_cols(out + k * w.d, acc, col, w.d, whole);
        } else {
            const f32x4 mine = chain(ts, links, wave * SLOTS + slot, WAVES * SLOTS);
            if (slot == 0) share[wave][lane] = mine;
            __syncthreads();
            if (wave == 0 && slot == 0 && live) {
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < WAVES; ++j) acc += share[j][lane];
                store_cols(out + k * w.d, acc, col, w.d, whole);
            }
            __syncthreads();
        }
    }
}

// list[0 .. count) of 256 threads, in the order of its codes k0 .. k0 + 2^bits - 1; entries of one code stay in theirs.  Stable counting
// passes of up to 8 bits: a wave has a quarter of the list, E entries a lane in registers, lanes of equal digit find each other by
// one ballot a bit, and what the waves have of a digit lies in the order of the waves.  (A bitonic sort in LDS took 30 us for 4096
// entries, this one 3 a pass.)  scratch: 4 KB, wave_sum: 4 numbers.
template <int E>
__device__ __forceinline__ void sort_list(CodePair* list, int count, uint32_t k0, int bits, f32x4* scratch, int* wave_sum) {
    uint32_t* at = reinterpret_cast<uint32_t*>(scratch);   // (4 waves, 256 digits)
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t* mine = at + wave * 256;
    const int rounds = (count + 255) / 256, i0 = wave * rounds * 64 + lane;
    for (int shift = 0; shift < bits; shift += 8) {
        const int width = bits - shift < 8 ? bits - shift : 8;
        __syncthreads();                                   // (behind the list's and the scratch's last use)
#pragma unroll
        for (int w = 0; w < 4; ++w) at[w * 256 + tid] = 0;
        __syncthreads();
        CodePair held[E];
        uint32_t rank[E];
#pragma unroll
        for (int r = 0; r < E; ++r) {
            rank[r] = 0;
            if (r < rounds) {                              // (uniform)
                const bool in = i0 + r * 64 < count;
                held[r] = list[in ? i0 + r * 64 : 0];
                const uint32_t digit = ((held[r].code - k0) >> shift) & 255u;
                uint64_t same = __ballot(in);
                for (int b = 0; b < width; ++b) {
                    const uint64_t set = __ballot((digit >> b) & 1);
                    same &= (digit >> b) & 1 ? set : ~set;
                }
                if (in) {
                    const uint32_t below = __popcll(same & ((1ull << lane) - 1));
                    // (all lanes read before the first of them writes: LDS operations of a wave stay in order)
                    const uint32_t before = __hip_atomic_load(&mine[digit], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
                    if (below == 0) __hip_atomic_store(&mine[digit], before + (uint32_t)__popcll(same), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
                    rank[r] = before + below;
                }
            }
        }
        __syncthreads();
        // a thread a digit: where its entries start, for each wave
        uint32_t n[4], total = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            n[w] = at[w * 256 + tid];
            total += n[w];
        }
        uint32_t scan = total;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t up = (uint32_t)__shfl_up((int)scan, o, 64);
            if (lane >= o) scan += up;
        }
        if (lane == 63) wave_sum[wave] = (int)scan;
        __syncthreads();
        uint32_t start = scan - total;
        for (int w = 0; w < wave; ++w) start += (uint32_t)wave_sum[w];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            at[w * 256 + tid] = start;
            start += n[w];
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < E; ++r) {
            if (r < rounds && i0 + r * 64 < count) list[mine[((held[r].code - k0) >> shift) & 255u] + rank[r]] = held[r];
        }
    }
    __syncthreads();
}

// All in one for few rows: the workgroup's codes are [k0, k0 + codes).  Its rows come out of the indices in row order, eight
// indices a thread at a time, and are put in the order of their codes: by a bitonic sort of (code, row) in registers where they
// are few (256, a thread each), by sort_list where they are more.  Groups of lanes then walk the codes, several to a code where
// there are more groups than codes; runs of more than kRun rows are walked by all the groups together, one run after the other.
// Of up to kFew codes with many rows, everybody walks the unsorted list once for each code, which is cheaper than the sort (2048
// rows, 8 x 256 x 128, two codes a workgroup, 40 % of the rows on one code, gradient of a lookup: 27 us, 30 sorted) and dearer with
// more codes (4096 rows, 150000 x 32, 147 codes a workgroup, 300 neighbouring codes in use: 700 us, 39 sorted).  The last workgroup
// has the rows without a code too, where rows have an output of their own.
template <class Op, int LPR, int CAP>                     // CAP: most rows, a power of two
__global__ __launch_bounds__(256) void code_small_kernel(const Op op, const IndexView index, float* __restrict__ out_all, int rows,
                                                        uint32_t K, int d, int codes) {
    constexpr int SLOTS = 256 / LPR, PER = 8, FLIGHT = Op::kOwn ? 4 : 8, kRun = 64, kFew = 4;
    __shared__ CodePair list[CAP];
    __shared__ f32x4 share[256];
    __shared__ int wave_count[PER][4], runs, run_at[CAP / kRun];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, slot = tid / LPR;
    const int p = blockIdx.y, col = (int)blockIdx.z * 256 + (tid % LPR) * 4;
    const bool live = col < d, whole = (d & 3) == 0;
    const uint32_t k0 = blockIdx.x * (uint32_t)codes;
    const uint32_t kend = k0 + codes < K ? k0 + codes : K;
    const uint32_t k1 = Op::kOwn && blockIdx.x == gridDim.x - 1 ? K + 1 : kend;
    int count = 0;
    for (int r0 = 0; r0 < rows; r0 += 256 * PER) {
        uint32_t k[PER];
        uint64_t m[PER];
        codes_at<PER>(index, p, r0 + tid, 256, rows, K, k);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (r0 + j * 256 + tid >= rows) k[j] = k1;
            m[j] = __ballot(k[j] >= k0 && k[j] < k1);
            if (lane == 0) wave_count[j][wave] = __popcll(m[j]);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            int at = count;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i < wave) at += wave_count[j][i];
                count += wave_count[j][i];
            }
            if (k[j] >= k0 && k[j] < k1) list[at + __popcll(m[j] & ((1ull << lane) - 1))] = CodePair{k[j], (uint32_t)(r0 + j * 256 + tid)};
        }
        __syncthreads();
    }
    float* out = out_all + (int64_t)p * K * d + col;
    const bool sums = out_all != nullptr;
    auto sum_range = [&](auto flight, int lo, int hi) {
        constexpr int F = decltype(flight)::value;         // rows in flight
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int j = lo; j < hi; j += F) {
            typename Op::Row row[F];
            f32x4 v[F];
#pragma unroll
            for (int i = 0; i < F; ++i) row[i] = op.template load<false>(list[j + i < hi ? j + i : hi - 1], p, live ? col : 0);
#pragma unroll
            for (int i = 0; i < F; ++i) v[i] = op.value(row[i]);
#pragma unroll
            for (int i = 0; i < F; ++i)
                if (j + i < hi) {
                    acc += v[i];
                    op.template own<false>(row[i], list[j + i].row, p, col);
                }
        }
        return acc;
    };
    // the sum of every group's share of a code's rows, written (called by the whole workgroup)
    auto store_joined = [&](uint32_t k, f32x4 acc) {
#pragma unroll
        for (int o = 32; o >= LPR; o >>= 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], o, 64);
        if (lane < LPR) share[wave * LPR + lane] = acc;
        __syncthreads();
        if (tid < LPR && live) {
            for (int w = 1; w < 4; ++w) acc += share[w * LPR + tid];
            store_cols(out + (int64_t)k * d, acc, col, d, whole);
        }
        __syncthreads();
    };
    const int n = (int)(k1 - k0);
    if (__builtin_expect(count > 256 && n <= kFew, 0)) {
        const int lo = count * slot / SLOTS, hi = count * (slot + 1) / SLOTS;
        for (uint32_t k = k0; k < k1; ++k) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            for (int j = lo; j < hi; j += FLIGHT) {
                CodePair pr[FLIGHT];
                bool any = false;
#pragma unroll
                for (int i = 0; i < FLIGHT; ++i) {
                    pr[i] = list[j + i < hi ? j + i : hi - 1];
                    any |= pr[i].code == k;
                }
                if (!any) continue;
                typename Op::Row row[FLIGHT];
#pragma unroll
                for (int i = 0; i < FLIGHT; ++i) row[i] = op.template load<false>(pr[i], p, live ? col : 0);
#pragma unroll
                for (int i = 0; i < FLIGHT; ++i) {
                    const f32x4 v = op.value(row[i]);
                    if (j + i < hi && pr[i].code == k) {
                        acc += v;
                        op.template own<false>(row[i], pr[i].row, p, col);
                    }
                }
            }
            if (sums && k < kend) store_joined(k, acc);    // (uniform)
        }
        return;
    }
    auto key_of = [](const CodePair& at) { return (uint64_t)at.code << 32 | at.row; };
    auto first_of = [&](uint32_t k) {                      // the first entry whose code is not below k
        int lo = 0, hi = count;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (list[mid].code < k) lo = mid + 1;
            else hi = mid;
        }
        return lo;
    };
    if (__builtin_expect(count <= 256, 1)) {
        uint64_t key = tid < count ? key_of(list[tid]) : ~0ull;
        for (int width = 2; width <= 256; width *= 2) {
            if (width / 2 >= count) break;                 // (uniform: everything behind `count` is the largest key already)
            for (int step = width / 2; step > 0; step /= 2) {
                uint64_t other;
                if (step < 64) other = (uint64_t)__shfl_xor((long long)key, step, 64);
                else {
                    uint64_t* keys = reinterpret_cast<uint64_t*>(share);
                    keys[tid] = key;
                    __syncthreads();
                    other = keys[tid ^ step];
                    __syncthreads();
                }
                const bool up = (tid & width) == 0, low = (tid & step) == 0;
                key = (up == low) == (key < other) ? key : other;
            }
        }
        if (tid < count) list[tid] = CodePair{(uint32_t)(key >> 32), (uint32_t)key};
        __syncthreads();
    } else {
        bool other = false;
        for (int j = tid; j < count; j += 256) other |= list[j].code != list[0].code;
        if (__syncthreads_or(other)) sort_list<CAP / 256>(list, count, k0, 32 - __clz(n - 1), share, wave_count[0]);
    }
    // the long runs of a workgroup that may have some
    const bool many = n > kFew && count > kRun;
    if (__builtin_expect(many, 0)) {
        if (tid == 0) runs = 0;
        __syncthreads();
        for (int j = tid; j + kRun < count; j += 256)      // (in any order: every run has a sum of its own)
            if (list[j + kRun].code == list[j].code && (j == 0 || list[j - 1].code != list[j].code)) run_at[atomicAdd(&runs, 1)] = j;
        __syncthreads();
    }
    const int parts = n < SLOTS ? SLOTS / n : 1;           // groups that share a code
    for (int c0 = 0; c0 < n; c0 += SLOTS / parts) {
        const int c = c0 + slot / parts, part = slot % parts;
        bool mine = slot / parts < SLOTS / parts && c < n;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        if (mine) {
            const int lo = first_of(k0 + c), len = first_of(k0 + c + 1) - lo;
            mine = !many || len <= kRun;
            if (mine) acc = sum_range(std::integral_constant<int, 4>(), lo + len * part / parts, lo + len * (part + 1) / parts);
        }
        if (!sums) continue;
        if (parts > 1) {                                   // (then there is one round)
            share[tid] = acc;
            __syncthreads();
            if (mine && part == 0)
                for (int j = 1; j < parts; ++j) acc += share[tid + j * LPR];
        }
        if (mine && part == 0 && live && k0 + c < kend) store_cols(out + (int64_t)(k0 + c) * d, acc, col, d, whole);
    }
    if (__builtin_expect(!many, 1)) return;
    __syncthreads();                                       // (behind the readers of share)
    for (int i = 0; i < runs; ++i) {
        const int lo = run_at[i];
        const uint32_t k = list[lo].code;
        const int len = first_of(k + 1) - lo;
        const f32x4 acc = sum_range(std::integral_constant<int, FLIGHT>(), lo + len * slot / SLOTS, lo + len * (slot + 1) / SLOTS);
        if (sums && k < kend) store_joined(k, acc);        // (uniform)
    }
}

template <class Op, int LPR>
int walk_launch_lpr(const Op& op, const SortPlan& s, const IndexView& index, char* ws, float* out, int d, hipStream_t stream) {
    const unsigned cchunks = (unsigned)((d + 255) / 256);
    if (s.passes == 0) {
        // codes a workgroup: about a thousand workgroups
        int64_t codes = ((int64_t)s.K * s.num_pq + 1023) / 1024;
        if (codes < 1) codes = 1;
        const unsigned gx = (unsigned)(((int64_t)s.K + codes - 1) / codes);
        const dim3 grid(gx, s.num_pq, cchunks);
        if (s.rows <= kSmallRows / 2)
            hipLaunchKernelGGL((code_small_kernel<Op, LPR, kSmallRows / 2>), grid, dim3(256), 0, stream, op, index, out, (int)s.rows, s.K, d, (int)codes);
        else
            hipLaunchKernelGGL((code_small_kernel<Op, LPR, kSmallRows>), grid, dim3(256), 0, stream, op, index, out, (int)s.rows, s.K, d, (int)codes);
        return check_launch("code_small_kernel");
    }
    size_t at = 0;
    int rc = sort_launch(s, index, ws, &at, stream);
    if (rc != EQUSS_OK) return rc;
    WalkArgs w;
    w.pairs = reinterpret_cast<const CodePair*>(ws + at);
    w.starts = reinterpret_cast<const uint32_t*>(ws + s.starts);
    w.partial = reinterpret_cast<float*>(ws + s.partial);
    w.out = out; w.rows = s.rows; w.code0 = 0; w.tiles = s.tiles; w.tile = s.tile; w.d = d; w.dpad = (d + 3) / 4 * 4; w.K = s.K;
    constexpr int TILES_WG = 4 * (64 / LPR);
    const dim3 grid((unsigned)((s.tiles + TILES_WG - 1) / TILES_WG), s.num_pq, cchunks);
    if (s.tile == kTile) hipLaunchKernelGGL((code_accumulate_kernel<Op, LPR, 1>), grid, dim3(256), 0, stream, op, w);
    else hipLaunchKernelGGL((code_accumulate_kernel<Op, LPR, 2>), grid, dim3(256), 0, stream, op, w);
    rc = check_launch("code_accumulate_kernel");
    if (rc != EQUSS_OK || !out) return rc;
    if ((int64_t)s.K * s.num_pq <= 1024 && (int64_t)s.K * s.num_pq * cchunks <= 2048) hipLaunchKernelGGL((code_join_kernel<LPR, 16>), dim3(s.K, s.num_pq, cchunks), dim3(1024), 0, stream, w);
    else
        for (constexpr int64_t kMost = max_blocks(256) * 4; w.code0 < (int64_t)s.K; w.code0 += kMost) {   // (one launch below 67 million codes)
            const int64_t left = (int64_t)s.K - w.code0, codes = left < kMost ? left : kMost;
            hipLaunchKernelGGL((code_join_kernel<LPR, 4>), dim3((unsigned)((codes + 3) / 4), s.num_pq, cchunks), dim3(256), 0, stream, w);
        }
    return check_launch("code_join_kernel");
}

}  // namespace equss
