// The stable radix sort of (code, row) pairs behind the codeword sums: see code_sort.h.
#include "code_sort.h"

namespace {

using equss::CodePair;
using equss::IndexView;

// first pass: the indices themselves; later ones: the pairs of the pass before
struct Source {
    IndexView index;
    const CodePair* pairs;      // null in the first pass
    int64_t rows;
    uint32_t K;
};

// pairs i, i + step, ... (those past `end` give the last one)
template <int N>
__device__ __forceinline__ void pairs_at(const Source& s, int p, int64_t i, int step, int64_t end, CodePair (&out)[N]) {
    if (s.pairs) {
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = s.pairs[(int64_t)p * s.rows + (i + (int64_t)j * step < end ? i + (int64_t)j * step : end - 1)];
    } else {
        uint32_t code[N];
        equss::codes_at<N>(s.index, p, i, step, end, s.K, code);
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = CodePair{code[j], (uint32_t)(i + (int64_t)j * step)};
    }
}

__global__ __launch_bounds__(256) void code_count_kernel(const Source s, uint32_t* __restrict__ table, int chunk_rows, int shift, int bits) {
    __shared__ uint32_t hist[equss::kMaxBins];
    const int bins = 1 << bits, p = blockIdx.y, chunk = blockIdx.x, chunks = gridDim.x;
    for (int b = threadIdx.x; b < bins; b += 256) hist[b] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)chunk * chunk_rows, i1 = i0 + chunk_rows < s.rows ? i0 + chunk_rows : s.rows;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += 256 * 8) {
        CodePair pr[8];
        pairs_at<8>(s, p, i, 256, i1, pr);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j * 256 < i1) atomicAdd(&hist[(pr[j].code >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    uint32_t* row = table + ((int64_t)p * chunks + chunk) * bins;
    for (int b = threadIdx.x; b < bins; b += 256) row[b] = hist[b];
}

// A wave owns a quarter of the chunk, so that ranks follow the row order.  starts: (num_pq, K + 1), written by the last pass of
// one-pass sorts (whose bins are the codes), or null.  What this kernel waits for is latency, so loads come in batches: the
// wave's pairs eight times 64 at once (kept for the second look at them where that is all of them) and the chunks' counts
// up to 64 at once.
template <int PER>                                      // bins a thread: bins <= 256 PER
__global__ __launch_bounds__(256) void code_place_kernel(const Source s, const uint32_t* __restrict__ table, CodePair* __restrict__ dst,
                                                        uint32_t* __restrict__ starts, int chunk_rows, int shift, int bits) {
    constexpr int B = 8, NB = PER <= 2 ? 64 / PER : 16;
    __shared__ uint32_t base[4][256 * PER];             // next place of every bin, for each wave
    __shared__ uint32_t first[256 * PER];               // all of the bin's pairs, then where they start
    __shared__ uint32_t wave_sum[4];
    const int bins = 1 << bits, p = blockIdx.y, chunk = blockIdx.x, chunks = gridDim.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t i0 = (int64_t)chunk * chunk_rows + (int64_t)wave * (chunk_rows / 4);
    int64_t i1 = i0 + chunk_rows / 4;
    if (i1 > s.rows) i1 = s.rows;
    CodePair held[B];
    auto fetch = [&](int64_t i) __attribute__((always_inline)) { pairs_at<B>(s, p, i + lane, 64, i1, held); };
    if (i0 < i1) fetch(i0);
    const uint32_t* rows_p = table + (int64_t)p * chunks * bins;
    uint32_t before[PER], total[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) before[j] = total[j] = 0;
    // (bins is at least 2 and a power of two: a thread without a bin reads one of the others')
    const int at0 = tid & (bins - 1);
    for (int c0 = 0; c0 < chunks; c0 += NB) {
        uint32_t n[PER][NB];
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
            for (int i = 0; i < NB; ++i) n[j][i] = rows_p[(c0 + i < chunks ? c0 + i : chunks - 1) * bins + at0 + 256 * j];
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                before[j] += c0 + i < chunk ? n[j][i] : 0u;
                total[j] += c0 + i < chunks ? n[j][i] : 0u;
            }
    }
    if (tid >= bins) total[0] = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        first[tid + 256 * j] = total[j];
#pragma unroll
        for (int v = 0; v < 4; ++v) base[v][tid + 256 * j] = 0;
    }
    __syncthreads();
    for (int64_t i = i0; i < i1; i += 64 * B) {
        if (i != i0) fetch(i);
#pragma unroll
        for (int j = 0; j < B; ++j)
            if (i + j * 64 + lane < i1) atomicAdd(&base[wave][(held[j].code >> shift) & (bins - 1)], 1u);
    }
    // exclusive sum over the bins, PER consecutive ones a thread
    uint32_t sum = 0, mine[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        mine[j] = first[tid * PER + j];
        sum += mine[j];
    }
    uint32_t scan = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = (uint32_t)__shfl_up((int)scan, o, 64);
        if (lane >= o) scan += up;
    }
    if (lane == 63) wave_sum[wave] = scan;
    __syncthreads();
    uint32_t start = scan - sum;
    for (int i = 0; i < wave; ++i) start += wave_sum[i];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int b = tid * PER + j;
        first[b] = start;
        if (starts && chunk == 0 && (uint32_t)b <= s.K) starts[(int64_t)p * ((int64_t)s.K + 1) + b] = start;
        start += mine[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        uint32_t at = first[tid + 256 * j] + before[j];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const uint32_t n = base[v][tid + 256 * j];
            base[v][tid + 256 * j] = at;
            at += n;
        }
    }
    __syncthreads();
    // 64 pairs at a time: lanes of equal digit find each other by one ballot a bit; their rank is the number of such lanes below
    CodePair* out = dst + (int64_t)p * s.rows;
    if (i1 - i0 > 64 * B) fetch(i0);
    for (int64_t i = i0; i < i1; i += 64 * B) {
        if (i != i0) fetch(i);
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const bool in = i + j * 64 + lane < i1;
            const uint32_t digit = (held[j].code >> shift) & (bins - 1);
            uint64_t same = __ballot(in);
            for (int b = 0; b < bits; ++b) {
                const uint64_t set = __ballot((digit >> b) & 1);
                same &= (digit >> b) & 1 ? set : ~set;
            }
            if (in) {
                const uint32_t rank = __popcll(same & ((1ull << lane) - 1));
                // (all lanes read before the first of them writes: LDS operations of a wave stay in order)
                const uint32_t at = __hip_atomic_load(&base[wave][digit], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
                if (rank == 0) __hip_atomic_store(&base[wave][digit], at + (uint32_t)__popcll(same), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
                out[at + rank] = held[j];
            }
        }
    }
}

// where every code's run starts among the sorted pairs: the first pair whose code is not below it
__global__ __launch_bounds__(256) void code_runs_kernel(const CodePair* __restrict__ pairs, uint32_t* __restrict__ starts, int64_t rows, uint32_t K) {
    const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (k > (int64_t)K) return;
    const CodePair* pp = pairs + (int64_t)blockIdx.y * rows;
    int64_t lo = 0, hi = rows;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if ((int64_t)pp[mid].code < k) lo = mid + 1;
        else hi = mid;
    }
    starts[(int64_t)blockIdx.y * ((int64_t)K + 1) + k] = (uint32_t)lo;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

namespace equss {

bool sort_plan(SortPlan& s, int64_t rows, int num_pq, int64_t K, int d) {
    s = SortPlan{};
    s.rows = rows;
    s.num_pq = num_pq;
    s.K = (uint32_t)K;
    if (rows > 0x7fffff00 || num_pq > 65535 || K >= ((int64_t)1 << 31)) return false;
    int bits = 1;
    while (((int64_t)1 << bits) <= K) ++bits;              // values 0 .. K
    if (rows <= (bits > 11 ? kSmallRows : kSmallRows / 2)) return true;   // one kernel, no workspace
    s.passes = (bits + 10) / 11;
    for (int i = 0, left = bits; i < s.passes; ++i) {
        s.bits[i] = (left + s.passes - i - 1) / (s.passes - i);
        left -= s.bits[i];
    }
    int64_t chunk = (rows + 63) / 64;                      // at most 64 chunks: every one reads the others' counts
    if (chunk < 2048) chunk = 2048;
    s.chunk_rows = (int)((chunk + 255) / 256 * 256);
    s.chunks = (int)((rows + s.chunk_rows - 1) / s.chunk_rows);
    // tiles of 64, or as short as 8 where that leaves the chip half empty: 4096 waves
    const int64_t lanes = d >= 256 ? 64 : (d + 3) / 4;
    s.tile = kTile;
    while (s.tile > 8 && (rows + s.tile - 1) / s.tile * num_pq * lanes < 4096 * 64) s.tile /= 2;
    s.tiles = (rows + s.tile - 1) / s.tile;
    size_t at = 0;
    const size_t pairs = align256((size_t)num_pq * rows * sizeof(CodePair));
    s.pairs_a = at; at += pairs;
    s.pairs_b = at; at += s.passes > 1 ? pairs : 0;
    s.table = at; at += align256((size_t)num_pq * s.chunks * kMaxBins * sizeof(uint32_t));
    s.starts = at; at += align256((size_t)num_pq * (K + 1) * sizeof(uint32_t));
    s.partial = at; at += align256((size_t)num_pq * s.tiles * 2 * ((d + 3) / 4 * 4) * sizeof(float));
    s.total = at;
    return true;
}

int sort_launch(const SortPlan& s, const IndexView& index, char* ws, size_t* pairs_at, hipStream_t stream) {
    Source src;
    src.index = index; src.pairs = nullptr; src.rows = s.rows; src.K = s.K;
    uint32_t* table = reinterpret_cast<uint32_t*>(ws + s.table);
    uint32_t* starts = reinterpret_cast<uint32_t*>(ws + s.starts);
    const dim3 grid((unsigned)s.chunks, (unsigned)s.num_pq);
    size_t dst = s.pairs_a;
    int shift = 0;
    for (int i = 0; i < s.passes; ++i) {
        dst = (i & 1) ? s.pairs_b : s.pairs_a;
        hipLaunchKernelGGL(code_count_kernel, grid, dim3(256), 0, stream, src, table, s.chunk_rows, shift, s.bits[i]);
        int rc = check_launch("code_count_kernel");
        if (rc != EQUSS_OK) return rc;
        CodePair* to = reinterpret_cast<CodePair*>(ws + dst);
        uint32_t* runs = s.passes == 1 ? starts : nullptr;
        if (s.bits[i] <= 8) hipLaunchKernelGGL(code_place_kernel<1>, grid, dim3(256), 0, stream, src, table, to, runs, s.chunk_rows, shift, s.bits[i]);
        else if (s.bits[i] == 9) hipLaunchKernelGGL(code_place_kernel<2>, grid, dim3(256), 0, stream, src, table, to, runs, s.chunk_rows, shift, s.bits[i]);
        else if (s.bits[i] == 10) hipLaunchKernelGGL(code_place_kernel<4>, grid, dim3(256), 0, stream, src, table, to, runs, s.chunk_rows, shift, s.bits[i]);
        else hipLaunchKernelGGL(code_place_kernel<8>, grid, dim3(256), 0, stream, src, table, to, runs, s.chunk_rows, shift, s.bits[i]);
        rc = check_launch("code_place_kernel");
        if (rc != EQUSS_OK) return rc;
        shift += s.bits[i];
        src.pairs = reinterpret_cast<const CodePair*>(ws + dst);
    }
    *pairs_at = dst;
    if (s.passes > 1) {
        hipLaunchKernelGGL(code_runs_kernel, dim3((unsigned)(((int64_t)s.K + 1 + 255) / 256), (unsigned)s.num_pq), dim3(256), 0, stream, src.pairs, starts,
                           s.rows, s.K);
        return check_launch("code_runs_kernel");
    }
    return EQUSS_OK;
}

}  // namespace equss
