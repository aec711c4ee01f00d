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

constexpr int kCountThreads = 1024;

__global__ __launch_bounds__(kCountThreads) void code_count_kernel(const Source s, uint32_t* __restrict__ table, int chunk_rows, int shift, int bits) {
    __shared__ uint32_t hist[equss::kMaxBins];
    constexpr int B = 8;
    const int bins = 1 << bits, p = blockIdx.y, chunk = blockIdx.x, chunks = gridDim.x;
    for (int b = threadIdx.x; b < bins; b += kCountThreads) hist[b] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)chunk * chunk_rows, i1 = i0 + chunk_rows < s.rows ? i0 + chunk_rows : s.rows;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += kCountThreads * B) {
        CodePair pr[B];
        pairs_at<B>(s, p, i, kCountThreads, i1, pr);
#pragma unroll
        for (int j = 0; j < B; ++j)
            if (i + j * kCountThreads < i1) atomicAdd(&hist[(pr[j].code >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    uint32_t* row = table + ((int64_t)p * chunks + chunk) * bins;
    for (int b = threadIdx.x; b < bins; b += kCountThreads) row[b] = hist[b];
}

// Every wave owns a share of the chunk, so that ranks follow the row order.  starts: (num_pq, K + 1), written by the last pass of
// one-pass sorts (whose bins are the codes), or null.  What this kernel waits for is latency: a wave's pairs are loaded eight
// times 64 at once (and kept where that is all of them), the chunks' counts sixteen at once.  Many waves a workgroup make few
// chunks, i.e. few counts to read for each: 102400 rows, 8 sub-spaces, both kernels: 15.8 us with 16 waves and 15 chunks, 18.3 us
// with 4 waves and 50 chunks; two kernels that only launch and load take 9.  (Called over and over; in a lookup's gradient, with
// what else runs there in the caches, 17.7.)
template <int WAVES, int BINS>                          // bins <= BINS, a multiple or a fraction of the threads
__global__ __launch_bounds__(64 * WAVES) void code_place_kernel(const Source s, const uint32_t* __restrict__ table, CodePair* __restrict__ dst,
                                                               uint32_t* __restrict__ starts, int chunk_rows, int shift, int bits) {
    constexpr int B = 8, THREADS = 64 * WAVES, PER = BINS > THREADS ? BINS / THREADS : 1, NB = 16;
    __shared__ uint32_t base[WAVES][BINS];              // next place of every bin, for each wave
    __shared__ uint32_t first[PER * THREADS];           // all of the bin's pairs, then where they start
    __shared__ uint32_t wave_sum[WAVES];
    const int bins = 1 << bits, p = blockIdx.y, chunk = blockIdx.x, chunks = gridDim.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t i0 = (int64_t)chunk * chunk_rows + (int64_t)wave * (chunk_rows / WAVES);
    int64_t i1 = i0 + chunk_rows / WAVES;
    if (i1 > s.rows) i1 = s.rows;
    CodePair held[B];
    auto fetch = [&](int64_t i) __attribute__((always_inline)) { pairs_at<B>(s, p, i + lane, 64, i1, held); };
    if (i0 < i1) fetch(i0);
    const uint32_t* rows_p = table + (int64_t)p * chunks * bins;
    uint32_t before[PER], total[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) before[j] = total[j] = 0;
    if (tid < bins) {                                   // (with more than one bin a thread there are exactly PER)
        for (int c0 = 0; c0 < chunks; c0 += NB) {
            uint32_t n[PER][NB];
#pragma unroll
            for (int j = 0; j < PER; ++j)
#pragma unroll
                for (int i = 0; i < NB; ++i) n[j][i] = rows_p[(c0 + i < chunks ? c0 + i : chunks - 1) * bins + tid + THREADS * j];
#pragma unroll
            for (int j = 0; j < PER; ++j)
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    before[j] += c0 + i < chunk ? n[j][i] : 0u;
                    total[j] += c0 + i < chunks ? n[j][i] : 0u;
                }
        }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        first[tid + THREADS * j] = total[j];
        if (tid < BINS) {
#pragma unroll
            for (int v = 0; v < WAVES; ++v) base[v][tid + THREADS * j] = 0;
        }
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
        if (tid < BINS) {
            uint32_t at = first[tid + THREADS * j] + before[j], n[WAVES];
#pragma unroll
            for (int v = 0; v < WAVES; ++v) n[v] = base[v][tid + THREADS * j];
#pragma unroll
            for (int v = 0; v < WAVES; ++v) {
                base[v][tid + THREADS * j] = at;
                at += n[v];
            }
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
            uint64_t same = __ballot(in);
            if (same == 0) break;
            const uint32_t digit = (held[j].code >> shift) & (bins - 1);
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
    // chunks of up to 8192 rows, 512 for each of 16 waves, and shorter ones as long as there are no more than 16; at most 64 of
    // them in all: every one reads the others' counts
    int64_t chunk = (rows + 15) / 16;
    if (chunk > 8192) chunk = 8192;
    if (chunk < (rows + 63) / 64) chunk = (rows + 63) / 64;
    s.chunk_rows = (int)((chunk + 1023) / 1024 * 1024);
    s.chunks = (int)((rows + s.chunk_rows - 1) / s.chunk_rows);
    // tiles of 64, or as short as 8 where that leaves the chip half empty: 4096 waves, a wave for 256 columns (counted as one for
    // any wider row: 8192 rows, 4096 columns took 52 us, 37 with tiles of 32, and the partial sums 33 MB instead of 8)
    const int64_t lanes = (d + 3) / 4;
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
        hipLaunchKernelGGL(code_count_kernel, grid, dim3(kCountThreads), 0, stream, src, table, s.chunk_rows, shift, s.bits[i]);
        int rc = check_launch("code_count_kernel");
        if (rc != EQUSS_OK) return rc;
        CodePair* to = reinterpret_cast<CodePair*>(ws + dst);
        uint32_t* runs = s.passes == 1 ? starts : nullptr;
        if (s.bits[i] <= 9) hipLaunchKernelGGL((code_place_kernel<16, 512>), grid, dim3(1024), 0, stream, src, table, to, runs, s.chunk_rows, shift, s.bits[i]);
        else if (s.bits[i] == 10) hipLaunchKernelGGL((code_place_kernel<8, 1024>), grid, dim3(512), 0, stream, src, table, to, runs, s.chunk_rows, shift, s.bits[i]);
        else hipLaunchKernelGGL((code_place_kernel<4, 2048>), grid, dim3(256), 0, stream, src, table, to, runs, s.chunk_rows, shift, s.bits[i]);
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
