// Attention of sequences in groups that share their first pages (one instruction before many users' prompts, one prompt before many answers).
//
//   out[t, h] = (sum_shared 2^(s_j - M) v_j + sum_own 2^(s_j - M) v_j) / (sum_shared 2^(s_j - M) + sum_own 2^(s_j - M))
//
// Softmax sums over two sets of positions add up once both refer to the same maximum. The first set, the shared pages, is the same for all tokens of a group,
// whose rows (token, query head of a KV head) lie one after the other: for the kernels of paged_attn.cu and paged_attn_tc.cu a group is one sequence
// with all these rows and without new positions (kShared), so that its keys and values are read once and its rows fill the tensor cores' tiles. The second
// set, each sequence's own rows, is a sequence that starts behind its prefix (kOwn). Both leave sums, maximum and weighted values in f32, and the launch
// below joins them, a warp per (token, query head).
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "paged_attn.cuh"

namespace im {
namespace {

// One of the two sets as the join sees it.
struct PartSet {
    PagedAttn p;
    int rows;  // of a tile
    int tc;    // parts in the order of paged_attn_tc.cu, a NaN as the sum of weights of a row that has to be done again
};
struct PrefixJoin {
    PartSet shared, own;
    int group_new;
};

constexpr int kPjWarps = 8;

// Adds what the parts of row `r` of an item hold to a row's maximum, sum and columns lane * V .. of its values.
template <bool BF16, int HD, int MODE>
__device__ __forceinline__ void add_parts(const PartSet &s, int unit, int head, const PagedUnit &u, int r, float &M, float &L, float (&o)[HD / 32]) {
    constexpr int V = HD / 32;
    const PagedAttn &p = s.p;
    const int lane = threadIdx.x & 31, R = s.rows;
    const int2 span = *reinterpret_cast<const int2 *>(p.spans + 2 * ((long long)unit * p.kv.nkv + head));
    const bool whole = span.x >= p.whole_slot;
    const int c = span.x >> 1, parts = whole ? 1 : span.y - c + 1;
    auto slot = [&](int i) { return i == 0 ? (size_t)span.x : (size_t)(c + i) * 2; };
    for (int i0 = 0; i0 < parts; i0 += 32) {
        const float2 x = i0 + lane < parts ? p.part_ml[slot(i0 + lane) * R + r] : make_float2(-INFINITY, 0.0f);
        if (s.tc && __any_sync(0xffffffffu, x.y != x.y)) {  // not finite on the tensor cores: the whole row again, from the positions that it sees
            float y[V], m, l;
            plain_row<BF16, HD>(p, u, head, r, unit_from<MODE>(u), u.end, y, m, l);
            if (m == -INFINITY && l == 0.0f) return;
            const float top = fmaxf(M, m), f = ex2(m - top), corr = M == top ? 1.0f : ex2(M - top);
            M = top;
            L = L * corr + l * f;
#pragma unroll
            for (int j = 0; j < V; j++) {  // column lane * V + j lies with lane (lane * V + j) % 32
                float v = 0.0f;
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const float w = __shfl_sync(0xffffffffu, y[k], (lane * V + j) & 31);
                    if ((lane * V + j) / 32 == k) v = w;
                }
                o[j] = o[j] * corr + v * f;
            }
            return;
        }
        const float top = fmaxf(M, warp_max(x.x)), corr = M == top ? 1.0f : ex2(M - top);
        const float f = x.x == -INFINITY && x.y == 0.0f ? 0.0f : ex2(x.x - top);  // (nothing seen in this part)
        M = top;
        L = L * corr + warp_sum(x.y * f);
#pragma unroll
        for (int j = 0; j < V; j++) o[j] *= corr;
        const int m = min(32, parts - i0);
#pragma unroll 4
        for (int i = 0; i < m; i++) {
            const float g = __shfl_sync(0xffffffffu, f, i);
            const float *src = s.tc ? p.part_o + (slot(i0 + i) * (HD / 4) + lane * V / 4) * (R * 4) + r * 4 + lane * V % 4 : p.part_o + (slot(i0 + i) * R + r) * HD + lane * V;
            float v[V];
            if constexpr (V == 2) *reinterpret_cast<float2 *>(v) = *reinterpret_cast<const float2 *>(src);
            else
#pragma unroll
                for (int j = 0; j < V; j += 4) *reinterpret_cast<float4 *>(v + j) = *reinterpret_cast<const float4 *>(src + j);
#pragma unroll
            for (int j = 0; j < V; j++) o[j] += g == 0.0f ? 0.0f : v[j] * g;
        }
    }
}

template <bool BF16, int HD>
__global__ void __launch_bounds__(kPjWarps * 32) paged_prefix_join_kernel(const __grid_constant__ PrefixJoin a) {
    constexpr int V = HD / 32;
    pdl_trigger();
    pdl_wait();
    const PagedAttn &p = a.own.p;
    const int token = blockIdx.x, lane = threadIdx.x & 31, h = blockIdx.y * kPjWarps + (threadIdx.x >> 5);
    if (h >= p.group * p.kv.nkv || token < __ldg(p.start) || token >= __ldg(p.start + p.kv.nseq)) return;
    const int seq = paged_seq_of(p.start, p.kv.nseq, token), first = __ldg(p.start + seq), t = token - first;
    if (first < 0 || t < 0 || t >= p.max_new || __ldg(p.start + seq + 1) > p.tokens || token >= __ldg(p.start + seq + 1)) return;
    const int head = h / p.group, hq = h - head * p.group, group = paged_group_of(p, seq);
    float M = -INFINITY, L = 0.0f, o[V];
#pragma unroll
    for (int j = 0; j < V; j++) o[j] = 0.0f;
    if (group >= 0) {
        const long long place = (long long)token - __ldg(p.start + min(max(__ldg(p.group_start + group), 0), p.kv.nseq));
        if (place < 0 || place >= a.group_new) return;
        const int row = (int)place * p.group + hq, unit = group * a.shared.p.row_tiles + row / a.shared.rows, r = row % a.shared.rows;
        const PagedUnit u = paged_unit_of<kShared>(a.shared.p, unit, a.shared.rows);
        if (r < u.rows) add_parts<BF16, HD, kShared>(a.shared, unit, head, u, r, M, L, o);
    }
    const int row = t * p.group + hq, unit = seq * p.row_tiles + row / a.own.rows, r = row % a.own.rows;
    const PagedUnit u = paged_unit_of<kOwn>(p, unit, a.own.rows);
    if (r < u.rows && u.end > u.from) add_parts<BF16, HD, kOwn>(a.own, unit, head, u, r, M, L, o);
    const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
    uint32_t *dst = reinterpret_cast<uint32_t *>(p.out + token * p.os + (long long)h * HD + lane * V);
#pragma unroll
    for (int j = 0; j < V; j += 2) dst[j / 2] = pack16<BF16>(o[j] * inv, o[j + 1] * inv);
}

struct PartPlan {
    int rows, tile, row_tiles, units, ctas;
    size_t slots, bytes;
};
PartPlan part_plan(const Device *dev, int units, int nkv, int hd, long long rows) {
    PartPlan a;
    const int tc = paged_tc_rows(hd, rows);
    a.rows = tc ? tc : 16;
    a.tile = tc ? 128 : 64;
    a.row_tiles = (int)((rows + a.rows - 1) / a.rows);
    a.units = units * a.row_tiles;
    a.ctas = dev->sm_count * (tc || hd == 256 ? 1 : 2);
    const size_t items = (size_t)a.units * nkv;
    a.slots = ((size_t)a.ctas * 2 + items) * a.rows;
    a.bytes = a.slots * hd * 4 + a.slots * 8 + (items * 8 + 15) / 16 * 16;
    return a;
}

struct PrefixPlan {
    PartPlan shared, own;
    size_t bytes;
};
PrefixPlan prefix_plan(const Device *dev, const PagedView &v, int group, int max_new, int groups, int max_group_new) {
    PrefixPlan a;
    a.shared = part_plan(dev, groups, v.nkv, v.hd, (long long)max_group_new * group);
    a.own = part_plan(dev, v.nseq, v.nkv, v.hd, (long long)max_new * group);
    a.bytes = a.shared.bytes + a.own.bytes;
    return a;
}

int prefix_check(const im_paged_kv *kv, int num_heads, int num_groups, int max_group_new) {
    IM_REQUIRE(num_groups >= 0 && max_group_new >= 1, "%d groups of %d new tokens", num_groups, max_group_new);
    const long long tiles = ((long long)(num_heads / kv->num_kv_heads) * max_group_new + 15) / 16;
    IM_REQUIRE(tiles * std::max(num_groups, 1) * kv->num_kv_heads <= 1 << 24, "%d groups of %d new tokens are too many for one call", num_groups, max_group_new);
    return IM_OK;
}

// The launch's own: where its sums go, from `at` on.
unsigned char *lay_out(PagedAttn *p, const PartPlan &plan, int max_rows, unsigned char *at) {
    p->row_tiles = plan.row_tiles;
    const long long tiles = (long long)plan.units * p->kv.nkv * ((max_rows + (long long)plan.tile - 1) / plan.tile);
    p->ctas = (int)std::max(1ll, std::min<long long>(plan.ctas, tiles));
    p->whole_slot = 2 * plan.ctas;
    p->part_o = reinterpret_cast<float *>(at);
    p->part_ml = reinterpret_cast<float2 *>(p->part_o + plan.slots * p->kv.hd);
    p->spans = reinterpret_cast<int *>(p->part_ml + plan.slots);
    p->odd = nullptr;  // (rows of parts are marked in part_ml)
    return at + plan.bytes;
}

template <bool BF16, int HD>
int join(const PrefixJoin &a, int heads, cudaStream_t st) {
    IM_CUDA_CHECK(launch_k(paged_prefix_join_kernel<BF16, HD>, dim3((unsigned)a.own.p.tokens, (unsigned)((heads + kPjWarps - 1) / kPjWarps)), dim3(kPjWarps * 32), 0, st, a));
    return IM_OK;
}

}  // namespace
}  // namespace im

IM_EXPORT size_t im_cuda_paged_prefix_attention_scratch_bytes(const im_device *dev, const im_paged_kv *kv, int num_heads, int max_new, int num_groups, int max_group_new) {
    try {
        im::PagedView v;
        if (!dev || im::paged_view(kv, 0, &v) != IM_OK || im::attn_check(kv, num_heads, max_new) != IM_OK || im::prefix_check(kv, num_heads, num_groups, max_group_new) != IM_OK) return 0;
        return im::prefix_plan(dev, v, num_heads / v.nkv, max_new, num_groups, max_group_new).bytes;
    } catch (...) {
        return 0;
    }
}

IM_EXPORT int im_cuda_paged_prefix_attention(im_device *dev, const im_paged_kv *kv, int layer, const void *q_dev, int64_t q_stride, void *out_dev, int64_t out_stride,
                                             int num_heads, const int *token_start_dev, int num_tokens, int max_new, const int *group_start_dev, int num_groups,
                                             int max_group_new, const int *prefix_pages_dev, int max_prefix, const uint64_t *mask_dev, int mask_words, float scale, int max_len,
                                             void *scratch_dev, size_t scratch_bytes, void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    PrefixJoin a;
    PagedAttn &p = a.own.p;
    IM_REQUIRE(kv && kv->num_kv_heads > 0, "kv is NULL or has no heads");
    int rc = prefix_check(kv, num_heads, num_groups, max_group_new);
    if (rc != IM_OK) return rc;
    IM_REQUIRE(num_groups == 0 || (group_start_dev && prefix_pages_dev), "groups need their first sequences and numbers of shared pages");
    IM_REQUIRE(max_prefix >= 0, "max_prefix %d", max_prefix);
    bool empty;
    rc = attn_args(dev, kv, layer, q_dev, q_stride, out_dev, out_stride, num_heads, token_start_dev, num_tokens, max_new, mask_dev, mask_words, scale, max_len, &p, &empty);
    if (rc != IM_OK || empty) return rc;
    const PrefixPlan plan = prefix_plan(dev, p.kv, p.group, max_new, num_groups, max_group_new);
    IM_REQUIRE(scratch_dev && aligned16(scratch_dev) && scratch_bytes >= plan.bytes, "paged prefix attention needs %zu bytes of 16-byte aligned scratch (got %zu)", plan.bytes,
               scratch_dev ? scratch_bytes : (size_t)0);
    max_len = attn_length(p.kv, max_len);
    max_prefix = std::min(attn_length(p.kv, max_prefix), max_len);
    p.group_start = group_start_dev;
    p.prefix_pages = prefix_pages_dev;
    p.groups = num_groups;
    a.shared.p = p;
    a.shared.p.mask = nullptr;
    a.shared.p.max_new = max_group_new;
    a.group_new = max_group_new;
    unsigned char *at = lay_out(&a.shared.p, plan.shared, max_prefix, static_cast<unsigned char *>(scratch_dev));
    lay_out(&p, plan.own, max_len, at);
    a.shared.rows = plan.shared.rows;
    a.own.rows = plan.own.rows;
    a.shared.tc = plan.shared.rows > 16;
    a.own.tc = plan.own.rows > 16;
    const cudaStream_t st = as_stream(stream);
    const bool bf16 = kv->dtype == IM_DTYPE_BF16;
    const auto parts = [&](const PartSet &s, const PartPlan &q, int mode) {
        return s.tc ? paged_tc_part_launch(dev, s.p, bf16, mode, q.rows, q.units, st) : paged_part_launch(dev, s.p, bf16, mode, q.units, st);
    };
    if (num_groups > 0) rc = parts(a.shared, plan.shared, kShared);
    if (rc == IM_OK) rc = parts(a.own, plan.own, kOwn);
    if (rc != IM_OK) return rc;
#define IM_RUN(HD) (bf16 ? join<true, HD>(a, num_heads, st) : join<false, HD>(a, num_heads, st))
    switch (kv->head_dim) {
    case 64: return IM_RUN(64);
    case 128: return IM_RUN(128);
    default: return IM_RUN(256);
    }
#undef IM_RUN
    IM_GUARD_END
}
