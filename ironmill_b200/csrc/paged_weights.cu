// Attention that also adds up what every position of the cache is worth to the call's tokens: the sums by which an eviction chooses (paged_evict.cu).
//
//   out[t, h] = sum_j p_thj v_j,   sum[s, g, j] += sum over the new tokens t of s and the heads h of KV head g of p_thj,   p = softmax as in paged_attn.cu
//
// A weight is known once its row's maximum and sum over all positions are: the attention kernels leave both for every row, and a second look at the scores
// follows. Up to 16 rows of a KV head (single tokens) the scores themselves are kept, 4 bytes a row and position against 4 * head_dim of keys
// and values, and a position's thread adds up its rows' weights; short contexts do it in the attention's own launch. With more rows keeping the scores would
// cost more than the keys: they are computed again, transposed: positions in the rows of mma.sync's tiles, query rows in their columns, so that a position's sum
// stays in four lanes. Every position is one thread's (or four lanes') own: no atomics, and the same sums on every run.
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "paged_attn.cuh"

namespace im {
namespace {

constexpr int kSumThreads = 256;

// Sums from scores: a block takes kSumThreads positions of an item at a time.
template <bool BF16, int HD>
__global__ void __launch_bounds__(kSumThreads) paged_sum_kernel(const __grid_constant__ PagedAttn p) {
    constexpr int R = 16;
    __shared__ RowNorm norms[R];
    pdl_trigger();
    pdl_wait();
    const int item = blockIdx.x, unit = item / p.kv.nkv, head = item - unit * p.kv.nkv, tid = threadIdx.x;
    const PagedUnit u = paged_unit<R, kWeigh>(p, unit);
    if ((int)blockIdx.y * kSumThreads >= u.end) return;
    if (tid < u.rows) norms[tid] = RowNorm(p.stat[(long long)item * R + tid]);
    __syncthreads();
    const float *scores = p.scores + (long long)item * p.score_rows * p.score_cap;
    for (long long pos = (long long)blockIdx.y * kSumThreads + tid; pos < u.end; pos += (long long)gridDim.y * kSumThreads) {
        float v = 0.0f;
        if (pos >= p.score_cap) {
            v = plain_sum<BF16, HD>(p, u, head, (int)pos, norms);
        } else {
#pragma unroll 4
            for (int r = 0; r < u.rows; r++) v += norms[r].weight(scores[(long long)r * p.score_cap + pos]);
        }
        add_sum(p, u, head, (int)pos, v);
    }
}

// Sums from queries and keys: a block takes 128 positions of a sequence's KV head, 16 a warp, their keys in registers, and all of its rows, 64 at a time.
constexpr int kWeighThreads = 256, kWeighTile = 128, kWeighRows = 64;
template <int HD>
struct WeighShape {
    static constexpr int kKeys = kWeighTile * HD * 2, kRows = kWeighRows * HD * 2;
    static constexpr int kSmem = kKeys > 2 * kRows ? kKeys : 2 * kRows;  // the keys' place is the queries' once they are in registers
};

template <bool BF16, int HD>
__global__ void __launch_bounds__(kWeighThreads, HD == 256 ? 1 : 2) paged_weigh_kernel(const __grid_constant__ PagedAttn p, int R) {
    using S = WeighShape<HD>;
    constexpr int KS = HD / 16, CH = HD / 8, RPI = kWeighThreads / CH;
    extern __shared__ __align__(128) unsigned char weigh_smem[];
    __shared__ long long offs[kWeighTile];
    __shared__ RowNorm norms[2][kWeighRows];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seq = blockIdx.x / p.kv.nkv, head = blockIdx.x - seq * p.kv.nkv;
    const PagedUnit u = paged_unit_of<kWeigh>(p, seq * p.row_tiles, INT_MAX);  // all rows of the sequence
    const uint32_t smem = smem_u32(weigh_smem);
    const int c = tid % CH, r0 = tid / CH;  // a thread's 16 bytes of a row
    auto queries = [&](int row0, int buf) {  // 64 rows and their norms
#pragma unroll
        for (int i = 0; i < kWeighRows / RPI; i++) {
            const int r = i * RPI + r0, row = row0 + r;
            const bool there = row < u.rows;
            const int t = row / p.group, h = head * p.group + row - t * p.group;
            cp16(smem + buf * S::kRows + r * (HD * 2) + ((c ^ (r & 7)) << 4), p.q + (there ? (u.tok0 + t) * p.qs + (long long)h * HD + c * 8 : 0), there);
        }
        if (tid < kWeighRows) {
            const int row = row0 + tid, unit = seq * p.row_tiles + row / R;
            norms[buf][tid] = RowNorm(row < u.rows ? p.stat[((long long)unit * p.kv.nkv + head) * R + row % R] : make_float2(0.0f, 0.0f));
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (long long tile0 = (long long)blockIdx.y * kWeighTile; tile0 < u.end; tile0 += (long long)gridDim.y * kWeighTile) {
        const int p0 = (int)tile0;
        __syncthreads();  // the tile before is done
        if (tid < kWeighTile) offs[tid] = p0 + tid < u.end ? p.kv.row_of(seq, p0 + tid) : -1;
        __syncthreads();
        for (int r = r0; r < kWeighTile; r += RPI) {
            const long long at = offs[r];
            cp16(smem + r * (HD * 2) + ((c ^ (r & 7)) << 4), p.kc + (at < 0 ? 0 : at + (long long)head * p.kv.page * HD + c * 8), at >= 0);
        }
        asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        uint32_t kf[KS][4];
        {
            const int r = warp * 16 + (lane & 15);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) ldsm4(kf[ks], smem + r * (HD * 2) + (((2 * ks + (lane >> 4)) ^ (r & 7)) << 4));
        }
        __syncthreads();
        queries(0, 0);
        float sum[2] = {0.0f, 0.0f};
        const int chunks = (u.rows + kWeighRows - 1) / kWeighRows, pos = p0 + warp * 16 + (lane >> 2);
        for (int k = 0; k < chunks; k++) {
            if (k + 1 < chunks) queries((k + 1) * kWeighRows, (k + 1) & 1);
            else asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();
            const uint32_t qs = smem + (k & 1) * S::kRows;
            const bool edge = p0 + warp * 16 + 16 > u.len || (k + 1) * kWeighRows > u.rows;  // some row does not see some position, or is none
#pragma unroll 2
            for (int j = 0; j < kWeighRows / 8; j++) {
                if (k * kWeighRows + j * 8 >= u.rows) break;
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const int r = j * 8 + (lane & 7);
#pragma unroll
                for (int ks = 0; ks < KS; ks += 2) {
                    uint32_t b[4];
                    ldsm4(b, qs + r * (HD * 2) + (((2 * ks + (lane >> 3)) ^ (r & 7)) << 4));
                    mma16<BF16>(s, kf[ks], b[0], b[1]);
                    mma16<BF16>(s, kf[ks + 1], b[2], b[3]);
                }
                const int at = j * 8 + (lane & 3) * 2;
                const RowNorm a = norms[k & 1][at], b = norms[k & 1][at + 1];
                float w[4] = {a.weight(s[0] * p.scale2), b.weight(s[1] * p.scale2), a.weight(s[2] * p.scale2), b.weight(s[3] * p.scale2)};
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int row = k * kWeighRows + at + (i & 1), x = pos + (i >> 1) * 8;
                        if (row >= u.rows || x >= u.end || !paged_sees(p, u, row / p.group, x)) w[i] = 0.0f;
                    }
                }
                sum[0] += w[0] + w[1];
                sum[1] += w[2] + w[3];
            }
            __syncthreads();  // everyone has read the rows before others come in their place
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
            const int x = pos + i * 8;
            if ((lane & 3) == 0 && x < u.end) add_sum(p, u, head, x, offs[x - p0] < 0 ? 0.0f : sum[i]);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
}

// Room for scores: where there are up to 16 rows of a KV head and 256 MB hold them (32 sequences of 32 heads: 65536 positions).
constexpr size_t kScoreMost = (size_t)256 << 20;
struct WeighPlan {
    AttnPlan attn;
    int cap, rows;        // positions and rows of an item's scores, 0: none are kept
    size_t attn_bytes, stat_bytes, score_bytes;
    size_t used, bytes;   // by a call of this length, by any up to it
};
WeighPlan weigh_plan(const Device *dev, const PagedView &v, int group, int max_new, int max_len) {
    WeighPlan a;
    a.attn = attn_plan(dev, v.nseq, v.nkv, v.hd, group, max_new, max_len);
    const size_t items = (size_t)a.attn.units * v.nkv;
    a.attn_bytes = (a.attn.bytes + 15) / 16 * 16;
    a.stat_bytes = items * a.attn.rows * 8;
    a.rows = group * max_new;
    a.cap = 0;
    size_t most = 0;
    if (a.attn.rows == 16 && a.attn.row_tiles == 1 && items > 0) {
        const size_t of_tile = items * a.rows * 4 * 64, tiles = ((size_t)max_len + 63) / 64;
        most = std::min(tiles, kScoreMost / of_tile) * of_tile;
        if (tiles * of_tile <= kScoreMost) a.cap = (int)std::min<size_t>(tiles * 64, INT_MAX / 64 * 64);
    }
    a.score_bytes = a.cap ? most : 0;
    a.used = a.attn_bytes + a.stat_bytes + a.score_bytes;
    a.bytes = a.attn_bytes + a.stat_bytes + most;
    return a;
}

template <bool BF16, int HD>
int sums(const Device *dev, const PagedAttn &p, const WeighPlan &plan, int max_len, cudaStream_t st) {
    using S = WeighShape<HD>;
    static DeviceOnce once;
    if (once.first(dev->ordinal)) IM_CUDA_CHECK(cudaFuncSetAttribute((paged_weigh_kernel<BF16, HD>), cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    const auto blocks = [&](long long positions) { return (unsigned)std::max(1ll, std::min((max_len + positions - 1) / positions, 65535ll)); };
    if (p.scores)
        IM_CUDA_CHECK(launch_k(paged_sum_kernel<BF16, HD>, dim3((unsigned)(plan.attn.units * p.kv.nkv), blocks(kSumThreads)), dim3(kSumThreads), 0, st, p));
    else
        IM_CUDA_CHECK(launch_k(paged_weigh_kernel<BF16, HD>, dim3((unsigned)(p.kv.nseq * p.kv.nkv), blocks(kWeighTile)), dim3(kWeighThreads), (size_t)S::kSmem, st, p, plan.attn.rows));
    return IM_OK;
}

}  // namespace
}  // namespace im

IM_EXPORT size_t im_cuda_paged_attention_weights_scratch_bytes(const im_device *dev, const im_paged_kv *kv, int num_heads, int max_new, int max_len) {
    try {
        im::PagedView v;
        if (!dev || im::paged_view(kv, 0, &v) != IM_OK || im::attn_check(kv, num_heads, max_new) != IM_OK || max_len < 0) return 0;
        return im::weigh_plan(dev, v, num_heads / v.nkv, max_new, im::attn_length(v, max_len)).bytes;
    } catch (...) {
        return 0;
    }
}

IM_EXPORT int im_cuda_paged_attention_weights(im_device *dev, const im_paged_kv *kv, int layer, const void *q_dev, int64_t q_stride, void *out_dev, int64_t out_stride,
                                              int num_heads, const int *token_start_dev, int num_tokens, int max_new, const uint64_t *mask_dev, int mask_words, float scale,
                                              int max_len, float *weights_dev, int64_t seq_stride, int64_t head_stride, int rows, void *scratch_dev, size_t scratch_bytes,
                                              void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    PagedAttn p;
    bool empty;
    IM_REQUIRE(kv && kv->num_kv_heads > 0, "kv is NULL or has no heads");
    const int64_t most = (int64_t)1 << 40;
    IM_REQUIRE(rows >= 1 && head_stride >= rows && head_stride <= most && seq_stride <= most && head_stride <= most / kv->num_kv_heads &&
                   (kv->num_seqs <= 1 || seq_stride >= (kv->num_kv_heads - 1) * head_stride + rows),
               "sums of different sequences and heads overlap");
    int rc = attn_args(dev, kv, layer, q_dev, q_stride, out_dev, out_stride, num_heads, token_start_dev, num_tokens, max_new, mask_dev, mask_words, scale, max_len, &p, &empty);
    if (rc != IM_OK || empty) return rc;
    IM_REQUIRE(weights_dev && reinterpret_cast<uintptr_t>(weights_dev) % 4 == 0, "the sums are NULL or not 4-byte aligned");
    const long long span = 4 * ((kv->num_seqs - 1) * (long long)seq_stride + (kv->num_kv_heads - 1) * head_stride + rows), row = 2ll * num_heads * kv->head_dim;
    IM_REQUIRE(!share_memory(weights_dev, span, q_dev, 2 * (num_tokens - 1) * (long long)q_stride + row) && !share_memory(weights_dev, span, out_dev, 2 * (num_tokens - 1) * (long long)out_stride + row),
               "the sums lie over the queries or the outputs");
    max_len = attn_length(p.kv, max_len);
    const WeighPlan plan = weigh_plan(dev, p.kv, p.group, max_new, max_len);
    IM_REQUIRE(plan.used == 0 || (scratch_dev && aligned16(scratch_dev) && scratch_bytes >= plan.used), "paged attention with sums needs %zu bytes of 16-byte aligned scratch (got %zu)",
               plan.used, scratch_dev ? scratch_bytes : (size_t)0);
    attn_lay_out(&p, plan.attn, max_len, scratch_dev);
    unsigned char *at = static_cast<unsigned char *>(scratch_dev) + plan.attn_bytes;
    p.stat = reinterpret_cast<float2 *>(at);
    p.scores = plan.cap ? reinterpret_cast<float *>(at + plan.stat_bytes) : nullptr;
    p.score_cap = plan.cap;
    p.score_rows = plan.rows;
    p.sums = weights_dev;
    p.sum_seq = seq_stride;
    p.sum_head = head_stride;
    p.sum_cols = rows;
    const cudaStream_t st = as_stream(stream);
    const bool bf16 = kv->dtype == IM_DTYPE_BF16;
    rc = plan.attn.rows >= 128 ? paged_tc_weigh_launch(dev, p, bf16, plan.attn.rows, plan.attn.units, st) : paged_weigh_launch(dev, p, bf16, plan.attn.units, plan.attn.cluster, st);
    if (rc != IM_OK || (plan.attn.cluster && p.scores)) return rc;
#define IM_RUN(HD) (bf16 ? sums<true, HD>(dev, p, plan, max_len, st) : sums<false, HD>(dev, p, plan, max_len, st))
    switch (kv->head_dim) {
    case 64: return IM_RUN(64);
    case 128: return IM_RUN(128);
    default: return IM_RUN(256);
    }
#undef IM_RUN
    IM_GUARD_END
}
