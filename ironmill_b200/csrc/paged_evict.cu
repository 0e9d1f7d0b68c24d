// Eviction from a paged cache by accumulated weight.
//
// A sequence of n > budget rows keeps its last `recent` rows and, of the older ones, the H = budget - recent with the largest sums (ties: the lowest row), for
// every layer and KV head on its own. Kept rows below H stay where they are; the others come, in order, to the places of those that leave, and the recent rows
// behind them. That moves the fewest rows: closing up in order would move nearly all of them for one that leaves, and attention does not
// ask for their order (keys are rotated already). What order means something for, the recent rows, is kept.
//
// Two launches. The first finds the H-th largest sum of its (layer, sequence, head) by digits of 8 bits from the top, each a histogram in shared memory, walks the rows
// once more in order, and lists sources and targets. The second moves rows, a block per (layer, sequence, head) of the keys or the values. HBM bounds the second, the
// chain of passes over one list the first.
#include <limits.h>

#include <algorithm>

#include "paged.cuh"

namespace im {
namespace {

struct Evict {
    PagedView kv;
    const float *w;
    float *w_out;
    long long w_layer, w_seq, w_head, o_layer, o_seq, o_head;
    int budget, recent;
    int *len_out;
    int *count;  // [layers, sequences, heads]: moves
    int *moves;  // [layers, sequences, heads, 2, most]: targets, sources
    int most;
};

// Larger sums have larger keys; a NaN counts as the lowest, -0 as 0.
__device__ __forceinline__ uint32_t sum_key(float w) {
    if (w != w) w = -INFINITY;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int kEvThreads = 256, kEvWarps = kEvThreads / 32;

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

__global__ void __launch_bounds__(kEvThreads) paged_evict_select_kernel(const __grid_constant__ Evict a) {
    __shared__ int bins[kEvWarps][256];
    __shared__ int of_warp[kEvWarps];
    __shared__ int found[2];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, problem = blockIdx.x;
    const int head = problem % a.kv.nkv, seq = problem / a.kv.nkv % a.kv.nseq, layer = problem / a.kv.nkv / a.kv.nseq;
    const int n = a.kv.length(seq), H = a.budget - a.recent, old = n - a.recent;
    const float *w = a.w + layer * a.w_layer + seq * a.w_seq + head * a.w_head;
    float *out = a.w_out + layer * a.o_layer + seq * a.o_seq + head * a.o_head;
    if (layer == 0 && head == 0 && tid == 0) a.len_out[seq] = min(n, a.budget);
    if (n <= a.budget) {
        for (int i = tid; i < n; i += kEvThreads) out[i] = w[i];
        if (tid == 0) a.count[problem] = 0;
        return;
    }
    // ---- the H-th largest key, digit by digit; `above` of the others are larger
    uint32_t top = 0, mask = 0;
    int above = 0;
    for (int shift = 24; shift >= 0 && H > 0; shift -= 8) {
        for (int i = tid; i < kEvWarps * 256; i += kEvThreads) (&bins[0][0])[i] = 0;
        __syncthreads();
        for (int i = tid; i < old; i += kEvThreads) {
            const uint32_t k = sum_key(w[i]);
            if ((k & mask) == top) atomicAdd(&bins[warp][k >> shift & 255], 1);
        }
        __syncthreads();
        // thread t has digit 255 - t: counts from the top
        int mine = 0, total;
#pragma unroll
        for (int i = 0; i < kEvWarps; i++) mine += bins[i][255 - tid];
        const int before = above + block_before(mine, of_warp, total);
        if (before < H && before + mine >= H) found[0] = 255 - tid, found[1] = before;
        __syncthreads();
        top |= (uint32_t)found[0] << shift;
        mask |= 255u << shift;
        above = found[1];
        __syncthreads();
    }
    const int equal = H - above;  // so many of the rows with that key stay, the lowest
    // ---- in order of the rows: places that become free below H, rows that come from behind
    int *to = a.moves + (long long)problem * 2 * a.most, *from = to + a.most;
    int equals = 0, holes = 0, movers = 0;
    for (int r0 = 0; r0 < old && H > 0; r0 += kEvThreads) {
        const int r = r0 + tid;
        const float x = r < old ? w[r] : 0.0f;
        const uint32_t k = r < old ? sum_key(x) : 0;
        const bool same = r < old && k == top;
        int total;
        const int rank = equals + block_before(same, of_warp, total);
        equals += total;
        const bool stays = r < old && (k > top || (same && rank < equal));
        const bool hole = r < H && !stays, mover = r >= H && stays;
        const int place = block_before((hole ? 1 : 0) | (mover ? 1 << 16 : 0), of_warp, total);
        if (hole) to[holes + (place & 0xffff)] = r;
        if (mover) from[movers + (place >> 16)] = r;
        holes += total & 0xffff;
        movers += total >> 16;
        if (r < H && stays) out[r] = x;
    }
    __syncthreads();
    for (int i = tid; i < movers; i += kEvThreads) out[to[i]] = w[from[i]];
    for (int i = tid; i < a.recent; i += kEvThreads) out[H + i] = w[old + i];
    if (tid == 0) a.count[problem] = movers;
}

// A block per (layer, sequence, head) of keys or values. Sixteen bytes a lane; what comes from behind first (its sources lie from H on, its targets below), then the
// recent rows, a batch read before it is written: a target lies before its source, so no batch writes over what a later one reads.
constexpr int kMoveRows = 128;
__global__ void __launch_bounds__(kEvThreads) paged_evict_move_kernel(const __grid_constant__ Evict a, uint4 *kc, uint4 *vc) {
    __shared__ long long src[kMoveRows], dst[kMoveRows];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, problem = blockIdx.x;
    const int head = problem % a.kv.nkv, seq = problem / a.kv.nkv % a.kv.nseq, layer = problem / a.kv.nkv / a.kv.nseq;
    const int n = a.kv.length(seq), H = a.budget - a.recent, old = n - a.recent;
    if (n <= a.budget) return;
    const int words = a.kv.hd / 8;
    uint4 *base = (blockIdx.y ? vc : kc) + layer * (a.kv.layer_stride / 8) + (long long)head * a.kv.page * words;
    const int *to = a.moves + (long long)problem * 2 * a.most, *from = to + a.most;
    const int movers = a.count[problem], total = movers + a.recent;
    for (int i0 = 0; i0 < total;) {
        const int m = min(kMoveRows, (i0 < movers ? movers : total) - i0);
        if (tid < m) {
            const int i = i0 + tid;
            const long long f = a.kv.row_of(seq, i < movers ? from[i] : old + i - movers), t = a.kv.row_of(seq, i < movers ? to[i] : H + i - movers);
            src[tid] = t < 0 || f < 0 ? -1 : f / 8;
            dst[tid] = t / 8;
        }
        __syncthreads();
        const int pieces = m * words;
        for (int j0 = 0; j0 < kMoveRows * 32; j0 += kEvThreads * 8) {
            if (j0 >= pieces) break;
            uint4 x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int at = j0 + j * kEvThreads + tid;
                if (at < pieces && src[at / words] >= 0) x[j] = base[src[at / words] + at % words];
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int at = j0 + j * kEvThreads + tid;
                if (at < pieces && src[at / words] >= 0) base[dst[at / words] + at % words] = x[j];
            }
        }
        __syncthreads();
        i0 += m;
    }
}

struct EvictPlan {
    long long problems;
    int most;
    size_t bytes;
};
EvictPlan evict_plan(const PagedView &v, int budget, int recent) {
    EvictPlan a;
    a.problems = (long long)v.layers * v.nseq * v.nkv;
    a.most = (int)std::min<long long>(budget - recent, std::max(0, v.rows - budget));  // a mover leaves a place behind H, and every row from H on that stays has one before it
    a.bytes = (size_t)a.problems * 4 + (size_t)a.problems * 2 * a.most * 4;
    return a;
}

int evict_check(int budget, int recent) {
    IM_REQUIRE(budget >= 1 && recent >= 0 && recent <= budget, "a budget of %d rows, the last %d among them", budget, recent);
    return IM_OK;
}

}  // namespace
}  // namespace im

IM_EXPORT size_t im_cuda_paged_evict_scratch_bytes(const im_device *dev, const im_paged_kv *kv, int budget, int recent) {
    try {
        im::PagedView v;
        if (!dev || im::paged_view(kv, -1, &v) != IM_OK || im::evict_check(budget, recent) != IM_OK) return 0;
        return im::evict_plan(v, budget, recent).bytes;
    } catch (...) {
        return 0;
    }
}

IM_EXPORT int im_cuda_paged_evict(im_device *dev, const im_paged_kv *kv, const float *weights_dev, int64_t layer_stride, int64_t seq_stride, int64_t head_stride, int budget,
                                  int recent, float *weights_out_dev, int64_t out_layer_stride, int64_t out_seq_stride, int64_t out_head_stride, int *seq_len_out_dev,
                                  void *scratch_dev, size_t scratch_bytes, void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    Evict a;
    PagedView &v = a.kv;
    int rc = paged_view(kv, -1, &v);
    if (rc == IM_OK) rc = evict_check(budget, recent);
    if (rc != IM_OK) return rc;
    IM_REQUIRE(v.nseq == 0 || (weights_dev && weights_out_dev && seq_len_out_dev), "bad argument");
    const long long most = 1ll << 40;
    const auto apart = [&](int64_t layer, int64_t seq, int64_t head) {
        return head >= v.rows && head <= most / v.nkv && seq <= most && layer <= most && (v.nseq <= 1 || seq >= (v.nkv - 1) * head + v.rows) &&
               (v.layers == 1 || layer >= (std::max(v.nseq, 1) - 1) * seq + (v.nkv - 1) * head + v.rows) && layer <= most / v.layers && seq <= most / std::max(v.nseq, 1);
    };
    IM_REQUIRE(apart(layer_stride, seq_stride, head_stride) && apart(out_layer_stride, out_seq_stride, out_head_stride),
               "sums have a row for each of the page table's %d, those of different layers, sequences and heads apart", v.rows);
    const EvictPlan plan = evict_plan(v, budget, recent);
    IM_REQUIRE(plan.problems <= INT_MAX, "too many layers, sequences and heads");
    if (v.nseq > 0) {
        IM_REQUIRE(reinterpret_cast<uintptr_t>(weights_dev) % 4 == 0 && reinterpret_cast<uintptr_t>(weights_out_dev) % 4 == 0, "the sums are not 4-byte aligned");
        const auto span = [&](int64_t layer, int64_t seq, int64_t head) { return 4 * ((v.layers - 1) * layer + (v.nseq - 1) * seq + (v.nkv - 1) * head + v.rows); };
        const long long in = span(layer_stride, seq_stride, head_stride), out = span(out_layer_stride, out_seq_stride, out_head_stride), lens = 4ll * v.nseq,
                        table = 4 * ((v.nseq - 1) * v.table_stride + v.width);
        IM_REQUIRE(!share_memory(weights_out_dev, out, weights_dev, in) && !share_memory(weights_out_dev, out, v.len, lens) && !share_memory(weights_out_dev, out, v.table, table),
                   "the new sums lie over what is read");
        IM_REQUIRE(!share_memory(seq_len_out_dev, lens, weights_dev, in) && !share_memory(seq_len_out_dev, lens, v.len, lens) && !share_memory(seq_len_out_dev, lens, v.table, table) &&
                       !share_memory(seq_len_out_dev, lens, weights_out_dev, out),
                   "the new lengths lie over what is read or the new sums");
    }
    rc = paged_device(dev);
    if (rc != IM_OK) return rc;
    if (v.nseq == 0) return IM_OK;
    IM_REQUIRE(scratch_dev && aligned16(scratch_dev) && scratch_bytes >= plan.bytes, "eviction needs %zu bytes of 16-byte aligned scratch (got %zu)", plan.bytes,
               scratch_dev ? scratch_bytes : (size_t)0);
    a.w = weights_dev;
    a.w_out = weights_out_dev;
    a.w_layer = layer_stride; a.w_seq = seq_stride; a.w_head = head_stride;
    a.o_layer = out_layer_stride; a.o_seq = out_seq_stride; a.o_head = out_head_stride;
    a.budget = budget;
    a.recent = recent;
    a.len_out = seq_len_out_dev;
    a.count = static_cast<int *>(scratch_dev);
    a.moves = a.count + plan.problems;
    a.most = plan.most;
    const cudaStream_t st = as_stream(stream);
    IM_CUDA_CHECK(launch_k(paged_evict_select_kernel, dim3((unsigned)plan.problems), dim3(kEvThreads), 0, st, a));
    IM_CUDA_CHECK(launch_k(paged_evict_move_kernel, dim3((unsigned)plan.problems, 2), dim3(kEvThreads), 0, st, a, static_cast<uint4 *>(kv->k_dev), static_cast<uint4 *>(kv->v_dev)));
    return IM_OK;
    IM_GUARD_END
}
