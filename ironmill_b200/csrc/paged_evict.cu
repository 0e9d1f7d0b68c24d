// Eviction from a paged cache by accumulated weight.
//
// A sequence of n > budget rows keeps its last `recent` rows and, of the older ones, the H = budget - recent with the largest sums (ties: the lowest row), for
// every layer and KV head on its own. Kept rows below H stay where they are; the others come, in order, to the places of those that leave, and the recent rows
// behind them. That moves the fewest rows: closing up in order would move nearly all of them for one that leaves, and attention does not
// ask for their order (keys are rotated already). What order means something for, the recent rows, is kept.
//
// One launch, a block per (layer, sequence, head) and slice of the columns of keys and values. Every block finds the H-th largest sum for itself (the sums are 4 bytes beside 4 * head_dim
// of a row): by digits of 11 bits from the top, each a histogram in shared memory, the later ones of those keys alone that share the first; then one bit a row says whether it stays, and the i-th free place below H and the i-th row that
// comes from behind are found by their ranks among the bits. No lists, no scratch, nothing between blocks.
// 16 sequences of up to 4096 rows to 1024, 8 layers (434 MB moved in rows of 256 bytes): 104 us, of which choosing takes 18 (nothing to move) and moving, at HBM's rate for such rows, 5.6 TB/s, 78
// (rows that lie side by side: 8 TB/s, from L2 in part). One sequence of 28 layers, 1100 rows to 1000: 18 us, the chain of the choice's passes. In two launches with lists of moves between them 144 and 28 us.
#include <limits.h>

#include <algorithm>

#include "paged.cuh"

namespace im {
namespace {

struct Evict {
    PagedView kv;
    uint4 *kc, *vc;
    const float *w;
    float *w_out;
    long long w_layer, w_seq, w_head, o_layer, o_seq, o_head;
    int budget, recent;
    int *len_out;
    int cols;       // 16-byte columns of a slice, of a row's keys and values one after the other
    int bit_words;  // of 32 rows
};

// Larger sums have larger keys; a NaN counts as the lowest, -0 as 0.
__device__ __forceinline__ uint32_t sum_key(float w) {
    if (w != w) w = -INFINITY;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int kEvThreads = 256, kEvWarps = kEvThreads / 32;
constexpr int kListed = 1024;                   // keys that are picked out
constexpr int kMoveRows = 128, kMoveAhead = 8;  // rows of a batch; 16-byte pieces that a thread holds

// Sums of v over the threads before this one, the block's total in `total`.
__device__ __forceinline__ int block_before(int v, int *of_warp, int &total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == 31) of_warp[w] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kEvWarps; i++) {
        if (i < w) before += of_warp[i];
        total += of_warp[i];
    }
    return before + s - v;
}

// The position of the set (clear: not set) bit with `rank` such bits before it, among words [lo, hi); before[w]: bits set in the words before w.
__device__ __forceinline__ int nth_bit(const uint32_t *bits, const int *before, int lo, int hi, int rank, bool clear) {
    // the last word whose count before it is not above rank
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1, b = clear ? mid * 32 - before[mid] : before[mid];
        if (b <= rank) lo = mid;
        else hi = mid;
    }
    uint32_t word = clear ? ~bits[lo] : bits[lo];
    rank -= clear ? lo * 32 - before[lo] : before[lo];
    int at = lo * 32;
#pragma unroll
    for (int half = 16; half > 0; half >>= 1) {
        const int low = __popc(word & ((1u << half) - 1));
        if (rank >= low) rank -= low, word >>= half, at += half;
    }
    return at;
}

__global__ void __launch_bounds__(kEvThreads, 4) paged_evict_kernel(const __grid_constant__ Evict a) {
    extern __shared__ __align__(16) uint32_t ev_smem[];
    __shared__ __align__(16) int bins[2048];
    __shared__ uint32_t list[kListed];
    __shared__ int of_warp[kEvWarps];
    __shared__ int found[3];
    uint32_t *bits = ev_smem;                                              // [bit_words]: rows that stay
    int *before = reinterpret_cast<int *>(bits + a.bit_words);             // [bit_words + 1]: of them in the words before
    long long *src = reinterpret_cast<long long *>(bins), *dst = src + 2 * kMoveRows;  // (the histograms are done then)
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, problem = blockIdx.x, slice = blockIdx.y;
    const int head = problem % a.kv.nkv, seq = problem / a.kv.nkv % a.kv.nseq, layer = problem / a.kv.nkv / a.kv.nseq;
    const int n = a.kv.length(seq), H = a.budget - a.recent, old = n - a.recent;
    const float *w = a.w + layer * a.w_layer + seq * a.w_seq + head * a.w_head;
    float *out = a.w_out + layer * a.o_layer + seq * a.o_seq + head * a.o_head;
    if (layer == 0 && head == 0 && slice == 0 && tid == 0) a.len_out[seq] = min(n, a.budget);
    if (n <= a.budget) {
        if (slice == 0)
            for (int i = tid; i < n; i += kEvThreads) out[i] = w[i];
        return;
    }
    // ---- the H-th largest key, digit by digit from the top; `above` of the others are larger, `equals` are the same. Once few enough share the digits
    // found they are picked out, and the next digits are theirs; where all that share them stay, the rest of the key does not matter.
    uint32_t top = 0, mask = 0;
    int above = 0, equals = old, listed = -1;
    for (int digit = 0; digit < 3 && H > 0 && equals > H - above; digit++) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, count = digit < 2 ? 2048 : 1024;
        for (int i = 4 * tid; i < count; i += 4 * kEvThreads) *reinterpret_cast<int4 *>(bins + i) = make_int4(0, 0, 0, 0);
        if (listed < 0 && digit > 0 && equals <= kListed) {
            if (tid == 0) found[2] = 0;
            __syncthreads();
#pragma unroll 4
            for (int i = tid; i < old; i += kEvThreads) {
                const uint32_t k = sum_key(__ldg(w + i));
                if ((k & mask) == top) list[atomicAdd(&found[2], 1)] = k;
            }
            listed = equals;
        }
        __syncthreads();
        if (listed >= 0) {
            for (int i = tid; i < listed; i += kEvThreads)
                if ((list[i] & mask) == top) atomicAdd(&bins[list[i] >> shift & (count - 1)], 1);
        } else {
#pragma unroll 4
            for (int i = tid; i < old; i += kEvThreads) {
                const uint32_t k = sum_key(__ldg(w + i));
                if ((k & mask) == top) atomicAdd(&bins[k >> shift & (count - 1)], 1);
            }
        }
        __syncthreads();
        // a thread has `each` bins, the first one the highest
        const int each = count / kEvThreads;
        int mine = 0, sum;
        for (int i = 0; i < each; i++) mine += bins[count - 1 - tid * each - i];
        int larger = above + block_before(mine, of_warp, sum);
        if (larger < H && larger + mine >= H)
            for (int i = 0; i < each; i++) {
                const int bin = count - 1 - tid * each - i, n_bin = bins[bin];
                if (larger + n_bin >= H) {
                    found[0] = bin, found[1] = larger, found[2] = n_bin;
                    break;
                }
                larger += n_bin;
            }
        __syncthreads();
        top |= (uint32_t)found[0] << shift;
        mask |= (uint32_t)(count - 1) << shift;
        above = found[1];
        equals = found[2];
        __syncthreads();
    }
    // ---- which rows stay: larger keys, and of equal ones the lowest rows
    const int equal = H - above, words = (old + 31) / 32;
    int stay = 0;
    if (H == 0 || equals == equal) {
        for (int r0 = 0; r0 < words * 32; r0 += kEvThreads) {
            const int r = r0 + tid;
            const unsigned word = __ballot_sync(0xffffffffu, r < old && H > 0 && sum_key(__ldg(w + r)) >= top);
            if (lane == 0 && r / 32 < words) bits[r / 32] = word;
        }
    } else {
        int passed = 0;  // equal ones so far
        for (int r0 = 0; r0 < words * 32; r0 += kEvThreads) {
            const int r = r0 + tid;
            const uint32_t k = r < old ? sum_key(__ldg(w + r)) : 0;
            const bool same = r < old && k == top;
            int all;
            const int rank = passed + block_before(same, of_warp, all);
            passed += all;
            const unsigned word = __ballot_sync(0xffffffffu, (r < old && k > top) || (same && rank < equal));
            if (lane == 0 && r / 32 < words) bits[r / 32] = word;
        }
    }
    __syncthreads();
    for (int w0 = 0; w0 < words; w0 += kEvThreads) {
        int total;
        const int c = w0 + tid < words ? __popc(bits[w0 + tid]) : 0, b = stay + block_before(c, of_warp, total);
        if (w0 + tid < words) before[w0 + tid] = b;
        stay += total;
    }
    if (tid == 0) before[words] = stay;
    __syncthreads();
    const int low = H / 32, kept_below = before[low] + (H % 32 ? __popc(bits[low] & ((1u << (H % 32)) - 1)) : 0);  // (H < old: there is such a word, or before[words])
    const int movers = H - kept_below, total = movers + a.recent;
    // the i-th place that is free below H, and the i-th row from H on that stays
    auto hole = [&](int i) { return nth_bit(bits, before, 0, words, i, true); };
    auto mover = [&](int i) { return nth_bit(bits, before, 0, words, kept_below + i, false); };
    if (slice == 0) {
        for (int r = tid; r < H; r += kEvThreads)
            if (bits[r / 32] >> (r % 32) & 1) out[r] = w[r];
        for (int i = tid; i < movers; i += kEvThreads) out[hole(i)] = w[mover(i)];
        for (int i = tid; i < a.recent; i += kEvThreads) out[H + i] = w[old + i];
    }
    // ---- the rows: what comes from behind first (its sources lie from H on, its targets below), then the recent ones, a batch read before it is
    // written: a target lies before its source, so no batch writes over what a later one reads. The places of the next batch are looked up while one is on its way.
    const int per_row = a.kv.hd / 8, col0 = slice * a.cols, cols = min(a.cols, 2 * per_row - col0);
    const int step = kEvThreads / cols, row = tid / cols, col = col0 + tid - row * cols;  // rows that a turn of the threads covers
    uint4 *base = (col >= per_row ? a.vc + col - per_row : a.kc + col) + layer * (a.kv.layer_stride / 8) + (long long)head * a.kv.page * per_row;
    auto batch = [&](int i0) { return min(kMoveRows, (i0 < movers ? movers : total) - i0); };
    auto places = [&](int i0, int buf) {
        const int i = i0 + tid;
        if (tid >= batch(i0)) return;
        const long long f = a.kv.row_of(seq, i < movers ? mover(i) : old + i - movers), t = a.kv.row_of(seq, i < movers ? hole(i) : H + i - movers);
        src[buf * kMoveRows + tid] = t < 0 || f < 0 ? -1 : f / 8;
        dst[buf * kMoveRows + tid] = t / 8;
    };
    __syncthreads();
    if (total > 0) places(0, 0);
    __syncthreads();
    for (int i0 = 0, buf = 0; i0 < total; buf ^= 1) {
        const int m = batch(i0);
        const long long *from = src + buf * kMoveRows, *to = dst + buf * kMoveRows;
        for (int r0 = 0; r0 < m; r0 += step * kMoveAhead) {
            uint4 x[kMoveAhead];
#pragma unroll
            for (int j = 0; j < kMoveAhead; j++) {
                const int r = r0 + j * step + row;
                if (row < step && r < m && from[r] >= 0) x[j] = base[from[r]];
            }
            if (r0 == 0 && i0 + m < total) places(i0 + m, buf ^ 1);
            if (i0 >= movers) __syncthreads();
#pragma unroll
            for (int j = 0; j < kMoveAhead; j++) {
                const int r = r0 + j * step + row;
                if (row < step && r < m && from[r] >= 0) base[to[r]] = x[j];
            }
        }
        i0 += m;
        __syncthreads();
    }
}

int evict_check(int budget, int recent) {
    IM_REQUIRE(budget >= 1 && recent >= 0 && recent <= budget, "a budget of %d rows, the last %d among them", budget, recent);
    return IM_OK;
}

constexpr int kEvRows = 1 << 19;  // bits and counts of so many rows fit an SM's shared memory

}  // namespace
}  // namespace im

IM_EXPORT int im_cuda_paged_evict(im_device *dev, const im_paged_kv *kv, const im_paged_evict_args *args, void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    IM_REQUIRE(args, "args is NULL");
    const im_paged_evict_args &x = *args;
    Evict a;
    PagedView &v = a.kv;
    int rc = paged_view(kv, -1, &v);
    if (rc == IM_OK) rc = evict_check(x.budget, x.recent);
    if (rc != IM_OK) return rc;
    IM_REQUIRE(v.nseq == 0 || (x.weights_dev && x.weights_out_dev && x.seq_len_out_dev), "bad argument");
    IM_REQUIRE(v.rows <= kEvRows, "eviction takes page tables of up to %d rows (got %d)", kEvRows, v.rows);
    const long long most = 1ll << 40;
    const auto apart = [&](int64_t layer, int64_t seq, int64_t head) {
        return head >= v.rows && head <= most / v.nkv && seq <= most && layer <= most && (v.nseq <= 1 || seq >= (v.nkv - 1) * head + v.rows) &&
               (v.layers == 1 || layer >= (std::max(v.nseq, 1) - 1) * seq + (v.nkv - 1) * head + v.rows) && layer <= most / v.layers && seq <= most / std::max(v.nseq, 1);
    };
    IM_REQUIRE(apart(x.layer_stride, x.seq_stride, x.head_stride) && apart(x.out_layer_stride, x.out_seq_stride, x.out_head_stride),
               "sums have a row for each of the page table's %d, those of different layers, sequences and heads apart", v.rows);
    const long long problems = (long long)v.layers * v.nseq * v.nkv;
    IM_REQUIRE(problems <= INT_MAX, "too many layers, sequences and heads");
    if (v.nseq > 0) {
        IM_REQUIRE(reinterpret_cast<uintptr_t>(x.weights_dev) % 4 == 0 && reinterpret_cast<uintptr_t>(x.weights_out_dev) % 4 == 0, "the sums are not 4-byte aligned");
        const auto span = [&](int64_t layer, int64_t seq, int64_t head) { return 4 * ((v.layers - 1) * layer + (v.nseq - 1) * seq + (v.nkv - 1) * head + v.rows); };
        const long long in = span(x.layer_stride, x.seq_stride, x.head_stride), out = span(x.out_layer_stride, x.out_seq_stride, x.out_head_stride), lens = 4ll * v.nseq,
                        table = 4 * ((v.nseq - 1) * v.table_stride + v.width);
        IM_REQUIRE(!share_memory(x.weights_out_dev, out, x.weights_dev, in) && !share_memory(x.weights_out_dev, out, v.len, lens) && !share_memory(x.weights_out_dev, out, v.table, table),
                   "the new sums lie over what is read");
        IM_REQUIRE(!share_memory(x.seq_len_out_dev, lens, x.weights_dev, in) && !share_memory(x.seq_len_out_dev, lens, v.len, lens) && !share_memory(x.seq_len_out_dev, lens, v.table, table) &&
                       !share_memory(x.seq_len_out_dev, lens, x.weights_out_dev, out),
                   "the new lengths lie over what is read or the new sums");
    }
    rc = paged_device(dev);
    if (rc != IM_OK) return rc;
    if (v.nseq == 0) return IM_OK;
    a.kc = static_cast<uint4 *>(kv->k_dev);
    a.vc = static_cast<uint4 *>(kv->v_dev);
    a.w = x.weights_dev;
    a.w_out = x.weights_out_dev;
    a.w_layer = x.layer_stride; a.w_seq = x.seq_stride; a.w_head = x.head_stride;
    a.o_layer = x.out_layer_stride; a.o_seq = x.out_seq_stride; a.o_head = x.out_head_stride;
    a.budget = x.budget;
    a.recent = x.recent;
    a.len_out = x.seq_len_out_dev;
    // A block all of a row where there are many (layer, sequence, head), down to 32 bytes of it where there are few
    const int per_row = v.hd / 8;
    a.cols = 2 * per_row;
    while (a.cols > 2 && problems * ((2 * per_row + a.cols - 1) / a.cols) < 3ll * dev->sm_count) a.cols = (a.cols + 1) / 2;
    const int slices = (2 * per_row + a.cols - 1) / a.cols;
    a.bit_words = (v.rows + 31) / 32;
    const size_t smem = (size_t)(2 * a.bit_words + 1) * 4;
    if (smem > 32768) {
        static DeviceOnce once;
        if (once.first(dev->ordinal)) IM_CUDA_CHECK(cudaFuncSetAttribute(paged_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (2 * (kEvRows / 32) + 1) * 4));
    }
    IM_CUDA_CHECK(launch_k(paged_evict_kernel, dim3((unsigned)problems, (unsigned)slices), dim3(kEvThreads), smem, as_stream(stream), a));
    return IM_OK;
    IM_GUARD_END
}
