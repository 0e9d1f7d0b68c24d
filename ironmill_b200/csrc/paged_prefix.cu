// Attention of sequences in groups that share their first pages (one instruction before many users' prompts, one prompt before many answers).
//
//   out[t, h] = (sum_shared 2^(s_j - M) v_j + sum_own 2^(s_j - M) v_j) / (sum_shared 2^(s_j - M) + sum_own 2^(s_j - M))
//
// Softmax sums over two sets of positions add up once both refer to the same maximum. The first set, the shared pages, is the same for all tokens of a group,
// whose rows (token, query head of a KV head) lie one after the other: a group is one sequence with all these rows and without new positions (kShared), so
// that its keys and values are read once for every 256 rows (every 16 of heads of 256) and its rows fill the tensor cores' tiles. The second set, each sequence's own rows, is a sequence that starts
// behind its prefix (kOwn). Both leave sums, maximum and weighted values in f32, and a last launch joins them.
//
// More than 16 rows of a unit go to paged_attn_tc.cu. Up to 16 rows (single tokens' own rows, small groups, heads of 256) are taken here, a chunk of 128 positions (64 for heads of 256) at a
// time, by CTAs that each have a few chunks of one item and end: several per SM in different phases hide the lookups, the loads' latency and the joining of
// warps behind each other's loads. (Equal shares of one list, as in paged_attn.cu, spend most of short items' time on their ends.) How many CTAs an item needs the host cannot
// know: where one sequence has far more rows of its own than the others, or is in no group, its items are longer than their CTAs' few chunks, and those items are left to equal
// shares of further CTAs, which look them up on the device.
// The launch for the own rows needs nothing of the one for the shared rows and starts beside it: kShared triggers its successor once everything before it is
// done, the successor does not wait at its start, and its first CTA waits at its end, so that the join finds both done.
//
// 64 sequences of up to 700 rows of their own behind 8192 (8.98 GFLOP, 132 MB): 52 us, of which the launches of both sets, side by side, 40 (58 SMs for the shared rows, 9 tiles of 128
// positions and 256 rows each; the others for the own rows, 3 TB/s) and the join 12, which is the latency of its three loads one after the other and 12 MB of parts from L2. 16 trees of 26
// nodes behind 30000 rows: 254 to 282 us in calls in a row, 730 to 810 TFLOP/s, by what the power cap leaves (240 us and 855 before it is reached), bound by the turns that the halves of a
// wide tile take (paged_attn_tc.cu). Heads of 64: 42 us for the first, 223 for the trees. Heads of 256 read the shared rows in tiles of 16 rows here, each tile all of them and a chunk only
// when the one before it is done: 230 us, and 3.5 ms for the trees, 6 and 14 times their floors.
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "paged_attn.cuh"

namespace im {
namespace {

// One of the two sets.
struct PartSet {
    PagedAttn p;
    int rows;    // of a tile
    int tc;      // by paged_attn_tc.cu: a NaN as the sum of weights of a row that has to be done again
    int chunks;  // else: CTAs, and so parts, of an item of up to `direct` chunks of positions; longer ones are cut into equal shares
    int direct, share_ctas;
    int units, cut_slot;  // slots from here on: two a CTA with a share (tc: from 0 on); items that one CTA had: their first own slot
};
struct PrefixJoin {
    PartSet shared, own;
    int group_new;
};

// ------------------------------------------------------------------------------------------------ up to 16 rows
constexpr int kPtWarps = 4, kPtThreads = kPtWarps * 32, kPtRows = 16;
template <int HD>
struct PtShape {
    static constexpr int kSlices = HD == 256 ? 1 : 2;          // of 16 positions, a warp's
    static constexpr int kChunk = kPtWarps * kSlices * 16;
    static constexpr int kPitch = HD + 8;                      // floats of a row of sums in shared memory
    static constexpr int kKeys = kSlices * 16 * HD * 2, kSums = kPtRows * kPitch * 4;
    static constexpr int kWarp = 2 * kKeys > kSums ? 2 * kKeys : kSums;  // sums take the place of keys and values
    static constexpr int kQ = kPtRows * HD * 2;                // queries, behind the warps' places
    static constexpr int kSmem = kPtWarps * kWarp + kQ;
};

// cp16 of keys and values: first to leave L2, where the parts are to stay until they are joined. (Also where several row tiles read the same rows, heads of 256: those are there for
// the tiles beside all the same; 64 sequences of 4 query heads a KV head behind 8192 rows 196.3 us so, 198.6 with the usual policy, 16 behind 30000 167.3 and 171.9.)
__device__ __forceinline__ uint64_t read_once() {
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ void cp16_once(uint32_t dst, const void *src, bool there, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0), "l"(policy) : "memory");
}

// Chunks k0, k0 + step, ... below k1 of an item, its part `slot`.
template <bool BF16, int HD, int MODE>
__device__ __forceinline__ void part_of_item(const PartSet &set, const PagedUnit &u, int head, int k0, int k1, int step, size_t slot, unsigned char *smem, long long (*offs)[32], float2 *ml,
                                             unsigned &bad_rows) {
    using S = PtShape<HD>;
    constexpr float kLift = BF16 ? 0.0f : 15.0f;  // fp16 weights: 2^15 at the row's maximum, as in paged_attn.cu
    constexpr int R = kPtRows, KS = HD / 16, NT = HD / 8, CH = HD / 8, SL = S::kSlices;
    const PagedAttn &p = set.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int from = unit_from<MODE>(u);
    unsigned char *mine = smem + warp * S::kWarp;
    const uint32_t ks_at = smem_u32(mine), vs_at = ks_at + S::kKeys;
    const uint64_t once = read_once();
    const uint32_t q_at = smem_u32(smem + kPtWarps * S::kWarp);
    for (int i = tid; i < R * CH; i += kPtThreads) {  // queries, on their way with the first keys
        const int r = i / CH, c8 = i % CH, row = u.row0 + r, t = row / p.group;
        cp16(q_at + r * (HD * 2) + ((c8 ^ (r & 7)) << 4), p.q + (r < u.rows ? (u.tok0 + t) * p.qs + (long long)(head * p.group + row - t * p.group) * HD + c8 * 8 : 0), r < u.rows);
    }
    int tok[2];
#pragma unroll
    for (int i = 0; i < 2; i++) tok[i] = (u.row0 + min((lane >> 2) + 8 * i, u.rows - 1)) / p.group;
    float m[2], l[2], o[NT][4];
#pragma unroll
    for (int i = 0; i < 2; i++) m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[n][j] = 0.0f;
    bool first = true;
    for (int k = k0; k < k1; k += step) {
        const int pos0 = from + k * S::kChunk + warp * (SL * 16);
        const int pos = pos0 + (lane & (SL * 16 - 1));
        const long long row = pos < u.end ? p.kv.row_of(u.seq, pos) : -1;
        const unsigned there = __ballot_sync(0xffffffffu, row >= 0);
        constexpr int RPI = 32 / CH > 0 ? 32 / CH : 1;  // rows of one request of the warp
        __syncwarp();  // the chunk before has been read
        if (lane < SL * 16) offs[warp][lane] = row < 0 ? -1 : row + (long long)head * p.kv.page * HD;
        __syncwarp();
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
#pragma unroll
            for (int i = 0; i < SL * 16 / RPI; i++) {
                const int r = i * RPI + (RPI > 1 ? lane / CH : 0), c8 = lane & (CH - 1);
                const long long at = offs[warp][r];
                cp16_once((kv ? vs_at : ks_at) + r * (HD * 2) + ((c8 ^ (r & 7)) << 4), (kv ? p.vc : p.kc) + (at < 0 ? 0 : at + c8 * 8), at >= 0, once);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        if (first) __syncthreads();  // everyone's queries
        else __syncwarp();
        first = false;
        float s[2 * SL][4];
#pragma unroll
        for (int n = 0; n < 2 * SL; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) s[n][j] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            uint32_t qf[4];
            ldsm4(qf, q_at + (lane & 15) * (HD * 2) + (((2 * ks + (lane >> 4)) ^ (lane & 7)) << 4));
#pragma unroll
            for (int sl = 0; sl < SL; sl++) {
                const int r = sl * 16 + (lane & 7) + ((lane >> 4) << 3), hi = (lane >> 3) & 1;
                uint32_t b[4];
                ldsm4(b, ks_at + r * (HD * 2) + (((2 * ks + hi) ^ (r & 7)) << 4));
                mma16<BF16>(s[2 * sl], qf, b[0], b[1]);
                mma16<BF16>(s[2 * sl + 1], qf, b[2], b[3]);
            }
        }
        const unsigned full = SL == 2 ? 0xffffffffu : 0xffffu;
        const bool part = (there & full) != full || (MODE == kOwn && pos0 + SL * 16 > u.len);  // some row may not see some position
#pragma unroll
        for (int n = 0; n < 2 * SL; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s[n][j] *= p.scale2;
                if (part) {
                    const int at = n * 8 + (lane & 3) * 2 + (j & 1);
                    if (!(there >> at & 1) || !paged_sees(p, u, tok[j >> 1], pos0 + at)) s[n][j] = -INFINITY;
                }
            }
        uint32_t w[SL][4], w2[SL][4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2 * SL; n++) top = fmaxf(top, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (__any_sync(0xffffffffu, top > m[i])) {
                const float m_new = fmaxf(m[i], top), corr = m_new == -INFINITY ? 1.0f : ex2(m[i] - m_new);
                m[i] = m_new;
                l[i] *= corr;
                if (k > k0)
#pragma unroll
                    for (int n = 0; n < NT; n++) o[n][2 * i] *= corr, o[n][2 * i + 1] *= corr;
            }
            const float base = m[i] == -INFINITY ? 0.0f : m[i] - kLift;
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < 2 * SL; n++) {  // weights as two 16-bit terms
                const float x0 = ex2(s[n][2 * i] - base), x1 = ex2(s[n][2 * i + 1] - base);
                sum += x0 + x1;
                const uint32_t x = pack16<BF16>(x0, x1);
                const float2 back = unpack16<BF16>(x);
                w[n / 2][2 * (n & 1) + i] = x;
                w2[n / 2][2 * (n & 1) + i] = pack16<BF16>(x0 - back.x, x1 - back.y);
            }
            l[i] += sum;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int sl = 0; sl < SL; sl++) {
            const int r = sl * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), hi = lane >> 4;
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                uint32_t b[4];
                ldsm4t(b, vs_at + r * (HD * 2) + (((n + hi) ^ (r & 7)) << 4));
                mma16<BF16>(o[n], w[sl], b[0], b[1]);
                mma16<BF16>(o[n + 1], w[sl], b[2], b[3]);
                mma16<BF16>(o[n], w2[sl], b[0], b[1]);
                mma16<BF16>(o[n + 1], w2[sl], b[2], b[3]);
            }
        }
    }
    // ---- four warps' sums joined, in order
#pragma unroll
    for (int i = 0; i < 2; i++) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if ((lane & 3) == 0) ml[warp * R + (lane >> 2) + 8 * i] = make_float2(m[i], l[i]);
    }
    __syncwarp();
    float *sums = reinterpret_cast<float *>(mine);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = (lane >> 2) + 8 * i;
        if (r < u.rows)
#pragma unroll
            for (int n = 0; n < NT; n++) *reinterpret_cast<float2 *>(sums + r * S::kPitch + n * 8 + (lane & 3) * 2) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
    }
    if (tid == 0) bad_rows = 0;
    __syncthreads();
    slot *= R;
    for (int i = tid; i < u.rows * (HD / 4); i += kPtThreads) {
        const int r = i / (HD / 4), d = i % (HD / 4) * 4;
        float M = -INFINITY, L = 0.0f, worst = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kPtWarps; k++) M = fmaxf(M, ml[k * R + r].x);
#pragma unroll
        for (int k = 0; k < kPtWarps; k++) {
            const float2 a = ml[k * R + r];
            const float4 v = *reinterpret_cast<const float4 *>(smem + k * S::kWarp + (r * S::kPitch + d) * 4);
            if (a.x == -INFINITY && a.y == 0.0f) {  // nothing seen: zeros, or zeros times something that is not finite
                continue;
            }
            const float f = ex2(a.x - M);
            L += a.y * f;
            x.x += v.x * f; x.y += v.y * f; x.z += v.z * f; x.w += v.w * f;
        }
        worst = x.x * 0.0f + x.y * 0.0f + x.z * 0.0f + x.w * 0.0f;
        if (worst != 0.0f) atomicOr(&bad_rows, 1u << r);
        *reinterpret_cast<float4 *>(p.part_o + (slot + r) * HD + d) = x;
        if (d == 0) p.part_ml[slot + r] = make_float2(M - kLift, L);  // (plain_row has no lift)
    }
    __syncthreads();
    if (const unsigned bad = bad_rows) {
        for (int r = warp; r < u.rows; r += kPtWarps) {
            if (!(bad >> r & 1)) continue;
            float M = -INFINITY, L = 0.0f, x[HD / 32];
#pragma unroll
            for (int i = 0; i < HD / 32; i++) x[i] = 0.0f;
            for (int k = k0; k < k1; k += step) {
                float y[HD / 32], m2, l2;
                plain_row<BF16, HD>(p, u, head, r, from + k * S::kChunk, min(from + (k + 1) * S::kChunk, u.end), y, m2, l2);
                if (m2 == -INFINITY && l2 == 0.0f) continue;
                const float top = fmaxf(M, m2), f = ex2(m2 - top), corr = M == top ? 1.0f : ex2(M - top);
                M = top;
                L = L * corr + l2 * f;
#pragma unroll
                for (int i = 0; i < HD / 32; i++) x[i] = x[i] * corr + y[i] * f;
            }
#pragma unroll
            for (int i = 0; i < HD / 32; i++) p.part_o[(slot + r) * HD + lane + 32 * i] = x[i];
            if (lane == 0) p.part_ml[slot + r] = make_float2(M, L);
        }
    }
}

// A CTA's share: where it is, what is left of it, and a unit that the threads look for.
struct PtShare {
    int unit, head, next, nth;
    long long left;
};
// Chunks c, c + chunks, ... of an item that is not long.
template <bool BF16, int HD, int MODE>
__device__ __forceinline__ void direct_part(const PartSet &set, int b, unsigned char *smem, long long (*offs)[32], float2 *ml, unsigned &bad_rows) {
    const PagedAttn &p = set.p;
    const int item = b / set.chunks, c = b - item * set.chunks, unit = item / p.kv.nkv, head = item - unit * p.kv.nkv;
    const PagedUnit u = paged_unit<kPtRows, MODE>(p, unit);
    const int all = unit_tiles<PtShape<HD>::kChunk, MODE>(u);
    if (c < all && all <= set.direct) part_of_item<BF16, HD, MODE>(set, u, head, c, all, set.chunks, (size_t)b, smem, offs, ml, bad_rows);
}

// An equal share of the list of the long items' chunks, item by item. (By itself: what it needs of registers is no cost of the kernel above. The share lies in shared memory.)
template <bool BF16, int HD, int MODE>
__device__ __noinline__ void share_parts(const PartSet &set, int cta, unsigned char *smem, long long (*offs)[32], float2 *ml, unsigned &bad_rows, PtShare &share) {
    constexpr int R = kPtRows, TILE = PtShape<HD>::kChunk;
    const PagedAttn &p = set.p;
    const int tid = threadIdx.x;
    PagedUnit u;
    const Share s = find_share<R, TILE, kPtThreads, MODE, true>(p, set.units, set.share_ctas, reinterpret_cast<long long *>(smem), u, set.direct, cta);
    if (s.from >= s.to) return;
    if (tid == 0) share = PtShare{s.unit, s.head, INT_MAX, 0, s.to - s.from};
    int head = s.head, k0 = s.tile;
    __syncthreads();
    for (;;) {
        const int all = unit_tiles<TILE, MODE>(u), item = share.unit * p.kv.nkv + head, k1 = (int)min((long long)all, k0 + share.left);
        const size_t slot = k0 == 0 && k1 == all ? (size_t)item * set.chunks : set.cut_slot + 2 * (size_t)cta + share.nth;
        int *span = p.spans + 2 * (long long)item;
        if (tid == 0 && k0 == 0) span[0] = (int)slot;
        if (tid == 0 && k1 == all) span[1] = cta;
        __syncthreads();
        if (tid == 0) share.left -= k1 - k0;
        part_of_item<BF16, HD, MODE>(set, u, head, k0, k1, 1, slot, smem, offs, ml, bad_rows);
        __syncthreads();
        if (share.left <= 0) return;
        // the next item: of the next head, or of the next long unit, which the threads look for together
        const int unit = share.unit;
        head = share.head + 1;
        k0 = 0;
        if (head == p.kv.nkv) {
            head = 0;
            for (int u0 = unit + 1; u0 < set.units; u0 += kPtThreads) {
                const int x = u0 + tid;
                if (x < set.units && unit_tiles<TILE, MODE>(paged_unit<R, MODE>(p, x)) > set.direct) atomicMin(&share.next, x);
                if (__syncthreads_or(share.next != INT_MAX)) break;
            }
            if (share.next == INT_MAX) return;
            u = paged_unit<R, MODE>(p, share.next);
        }
        const int next = head ? unit : share.next;
        __syncthreads();
        if (tid == 0) share = PtShare{next, head, INT_MAX, 1, share.left};
        __syncthreads();
    }
}

// CTAs, one set after the other: for items of the shared rows and of the own ones, then for shares of the long ones of either.
template <bool BF16, int HD>
__global__ void __launch_bounds__(kPtThreads, HD == 256 ? 2 : 3) paged_part_kernel(const __grid_constant__ PrefixJoin a, int shared_ctas, int own_ctas) {
    extern __shared__ __align__(128) unsigned char pt_smem[];
    __shared__ float2 ml[kPtWarps * kPtRows];
    __shared__ long long offs[kPtWarps][32];
    __shared__ unsigned bad_rows;
    __shared__ PtShare share;
    if (!a.own.p.early) pdl_wait();
    pdl_trigger();  // (the join looks up what this call was given before it waits)
    const int b = blockIdx.x, i = b - shared_ctas, cta = i - own_ctas, own_cta = shared_ctas ? cta - a.shared.share_ctas : cta;
    if (i < 0) direct_part<BF16, HD, kShared>(a.shared, b, pt_smem, offs, ml, bad_rows);
    else if (cta < 0) direct_part<BF16, HD, kOwn>(a.own, i, pt_smem, offs, ml, bad_rows);
    else if (own_cta < 0) share_parts<BF16, HD, kShared>(a.shared, cta, pt_smem, offs, ml, bad_rows, share);
    else share_parts<BF16, HD, kOwn>(a.own, own_cta, pt_smem, offs, ml, bad_rows, share);
    if (a.own.p.early && b == 0) pdl_wait();  // this launch ends after the one before it
}

// ------------------------------------------------------------------------------------------------ the join
// A block takes eight rows (token, query head of one KV head, token-major), a thread four columns of one: eight rows of a column quad lie side by side in the parts of
// paged_attn_tc.cu. What bounds it is the chain of lookups, so eight lanes find their rows' units before the launches in front of this one are done (those trigger it when
// everything before the call is), then places of parts, then 32 parts at a time of both sets: maxima and sums a lane each, factors to shared memory, values.
constexpr int kPjRows = 8, kPjParts = 32, kPjAhead = 6;
struct PjRow {
    int token;                // -1: not to be written
    long long out;
    int unit[2], r[2];        // shared, own: the unit (-1: no parts) and row of its tile
    int slot0[2], next[2], step[2], parts[2];  // slot of the first part, of the others less their steps; number of parts
};

template <int HD, int MODE>
__device__ __forceinline__ void find_unit(const PartSet &s, int unit, int r, PjRow &x) {
    constexpr int w = MODE == kOwn;
    const PagedUnit u = paged_unit_of<MODE>(s.p, unit, s.rows);
    const int from = unit_from<MODE>(u);
    if (r >= u.rows || u.end <= from) return;
    x.r[w] = r;
    x.unit[w] = unit;
    const int all = (u.end - from + PtShape<HD>::kChunk - 1) / PtShape<HD>::kChunk;
    x.parts[w] = s.tc || all > s.direct ? -1 : min(s.chunks, all);  // (-1: the spans say)
}
__device__ __forceinline__ void find_parts(const PartSet &s, int w, int head, PjRow &x) {
    if (x.unit[w] < 0) return;
    const long long item = (long long)x.unit[w] * s.p.kv.nkv + head;
    if (x.parts[w] < 0) {
        const int2 span = *reinterpret_cast<const int2 *>(s.p.spans + 2 * item);
        const int cta = (span.x - s.cut_slot) >> 1;
        const bool whole = s.tc ? span.x >= s.p.whole_slot : span.x < s.cut_slot;
        x.slot0[w] = span.x;
        x.next[w] = s.cut_slot + 2 * cta;
        x.step[w] = 2;
        x.parts[w] = whole ? 1 : span.y - cta + 1;
    } else {
        x.slot0[w] = x.next[w] = (int)(item * s.chunks);
        x.step[w] = 1;
    }
}
__device__ __forceinline__ size_t slot_of(int w, const PjRow &x, int part) { return part == 0 ? x.slot0[w] : x.next[w] + part * x.step[w]; }

template <bool BF16, int HD>
__global__ void __launch_bounds__(2 * HD) paged_prefix_join_kernel(const __grid_constant__ PrefixJoin a) {
    constexpr int V = HD / 32, kWarps = 2 * HD / 32;
    __shared__ PjRow rows[kPjRows];
    __shared__ float factor[kPjRows][kPjParts];
    __shared__ float2 state[kPjRows];  // maximum and sum so far
    __shared__ float corr[kPjRows];
    __shared__ float again[kPjRows][HD];
    __shared__ int most, odd;
    pdl_trigger();
    const PagedAttn &p = a.own.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, head = blockIdx.y;
    PjRow x;
    x.token = x.unit[0] = x.unit[1] = -1;
    x.parts[0] = x.parts[1] = 0;
    if (tid < kPjRows) {  // a lane per row
        const long long at = (long long)blockIdx.x * kPjRows + tid;
        const int token = (int)min(at / p.group, (long long)INT_MAX), hq = (int)(at - (long long)token * p.group);
        if (token < p.tokens && token >= __ldg(p.start) && token < __ldg(p.start + p.kv.nseq)) {
            int seq = 0;  // the last that starts at or before the token
            for (int hi = p.kv.nseq; hi - seq > 1;) {
                const int mid = (seq + hi) / 2;
                if (__ldg(p.start + mid) <= token) seq = mid;
                else hi = mid;
            }
            const int first = __ldg(p.start + seq), end = __ldg(p.start + seq + 1), t = token - first;
            if (first >= 0 && t >= 0 && t < p.max_new && end <= p.tokens && token < end) {
                const int group = paged_group_of(p, seq);
                const long long place = group < 0 ? 0 : (long long)token - __ldg(p.start + min(max(__ldg(p.group_start + group), 0), p.kv.nseq));
                if (place >= 0 && place < a.group_new) {
                    x.token = token;
                    x.out = token * p.os + (long long)(head * p.group + hq) * HD;
                    if (group >= 0) {
                        const int row = (int)place * p.group + hq, tile = row / a.shared.rows;
                        find_unit<HD, kShared>(a.shared, group * a.shared.p.row_tiles + tile, row - tile * a.shared.rows, x);
                    }
                    const int row = t * p.group + hq, tile = row / a.own.rows;
                    find_unit<HD, kOwn>(a.own, seq * p.row_tiles + tile, row - tile * a.own.rows, x);
                }
            }
        }
    }
    pdl_wait();
    if (tid < kPjRows) {
        find_parts(a.shared, 0, head, x);
        find_parts(a.own, 1, head, x);
        rows[tid] = x;
        state[tid] = make_float2(-INFINITY, 0.0f);
        const int n = __reduce_max_sync((1u << kPjRows) - 1, x.parts[0] + x.parts[1]);
        if (tid == 0) most = n, odd = 0;
    }
    __syncthreads();
    const int r = tid % kPjRows, q = tid / kPjRows;  // this thread's row and columns 4 q ..
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const size_t pitch0 = a.shared.tc ? (size_t)a.shared.rows * 4 : 4, pitch1 = a.own.tc ? (size_t)a.own.rows * 4 : 4;
    const float *base0 = a.shared.p.part_o + rows[r].r[0] * (a.shared.tc ? 4 : HD) + q * pitch0, *base1 = p.part_o + rows[r].r[1] * (a.own.tc ? 4 : HD) + q * pitch1;
    const int parts0 = rows[r].parts[0], parts = parts0 + rows[r].parts[1];
#pragma unroll 1
    for (int i0 = 0; i0 < most; i0 += kPjParts) {
        for (int i = warp; i < kPjRows; i += kWarps) {
            const PjRow &y = rows[i];
            const int part = i0 + lane, w = part >= y.parts[0], k = w ? part - y.parts[0] : part;
            const PartSet &s = w ? a.own : a.shared;
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (part < y.parts[0] + y.parts[1]) ml = s.p.part_ml[slot_of(w, y, k) * s.rows + y.r[w]];
            const bool redo = __any_sync(0xffffffffu, s.tc && ml.y != ml.y);  // not finite on the tensor cores: the row is done again below
            const float2 before = state[i];
            const float top = fmaxf(before.x, warp_max(ml.x)), c = before.x == top ? 1.0f : ex2(before.x - top);
            const float f = ml.x == -INFINITY && ml.y == 0.0f ? 0.0f : ex2(ml.x - top);  // (nothing seen in this part)
            const float l = before.y * c + warp_sum(ml.y * f);
            factor[i][lane] = f;
            __syncwarp();
            if (lane == 0) {
                state[i] = make_float2(top, l);
                corr[i] = c;
                if (redo) atomicOr(&odd, 1 << i);
            }
        }
        __syncthreads();
        const float c = corr[r];
        o = make_float4(o.x * c, o.y * c, o.z * c, o.w * c);
        const int n = min(parts - i0, kPjParts);
#pragma unroll 1
        for (int i = 0; i < n; i += kPjAhead) {  // requested together: one after the other they took a microsecond for two
            float4 v[kPjAhead];
#pragma unroll
            for (int j = 0; j < kPjAhead; j++) {
                const int part = i0 + min(i + j, n - 1);
                v[j] = *reinterpret_cast<const float4 *>(part < parts0 ? base0 + slot_of(0, rows[r], part) * a.shared.rows * HD
                                                                       : base1 + slot_of(1, rows[r], part - parts0) * a.own.rows * HD);
            }
#pragma unroll
            for (int j = 0; j < kPjAhead; j++) {
                const float f = i + j < n ? factor[r][i + j] : 0.0f;
                if (f != 0.0f) o.x += v[j].x * f, o.y += v[j].y * f, o.z += v[j].z * f, o.w += v[j].w * f;
            }
        }
        __syncthreads();
    }
    // ---- rows with sums on the tensor cores that are not finite: both sets again, from the positions that the row sees alone
    for (int w = 0; w < 2 && odd; w++) {
        for (int i = warp; i < kPjRows; i += kWarps) {
            if (!(odd >> i & 1)) continue;
            const float2 before = w ? state[i] : make_float2(-INFINITY, 0.0f);
            float y[V], m = -INFINITY, l = 0.0f;
            if (rows[i].unit[w] >= 0) {
                const PartSet &s = w ? a.own : a.shared;
                const PagedUnit u = w ? paged_unit_of<kOwn>(s.p, rows[i].unit[w], s.rows) : paged_unit_of<kShared>(s.p, rows[i].unit[w], s.rows);
                plain_row<BF16, HD>(s.p, u, head, rows[i].r[w], u.from, u.end, y, m, l);
#pragma unroll
                for (int j = 0; j < V; j++) again[i][lane + 32 * j] = y[j];
            }
            const float top = fmaxf(before.x, m), c = before.x == top ? 1.0f : ex2(before.x - top), f = m == -INFINITY && l == 0.0f ? 0.0f : ex2(m - top);
            __syncwarp();
            if (lane == 0) state[i] = make_float2(top, before.y * c + l * f), corr[i] = c, factor[i][0] = f;
        }
        __syncthreads();
        if (odd >> r & 1) {
            const float c = corr[r], f = factor[r][0];
            o = w ? make_float4(o.x * c, o.y * c, o.z * c, o.w * c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (f != 0.0f) o.x += again[r][4 * q] * f, o.y += again[r][4 * q + 1] * f, o.z += again[r][4 * q + 2] * f, o.w += again[r][4 * q + 3] * f;
        }
        __syncthreads();
    }
    if (rows[r].token < 0) return;
    const float L = state[r].y, inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
    *reinterpret_cast<uint2 *>(p.out + rows[r].out + 4 * q) = make_uint2(pack16<BF16>(o.x * inv, o.y * inv), pack16<BF16>(o.z * inv, o.w * inv));
}

// ------------------------------------------------------------------------------------------------ plans
struct PartPlan {
    int rows, row_tiles, units, tc;
    int ctas;          // with shares
    int most_chunks;   // not tcgen05: CTAs of an item
    size_t slots, spans;
    size_t bytes;
};
// tc: rows of a tile on tcgen05, 0: tiles of 16 here, with at most four CTAs an SM and at most one a chunk: more of them even out sequences of different lengths, but each
// leaves a part to join (32 sequences behind 4096 rows: 33 us with four, 37 with six, 40 with 24; 8 x 8 behind 3000: 53 with four or six, 57 with 24; 64 behind 8192: 53 with any).
// Items of more than kTurns chunks a CTA are cut into equal shares of further CTAs, two an SM (four users behind 30000 rows and one of 30000 by itself: 607 us without, 80 so; three an SM
// 83, and 73 instead of 70 for 63 users behind 8192; the number of turns, 4 to 32, makes no difference there, and up to 15 % either way for sequences that are all alike).
constexpr int kMostChunks = 64, kRounds = 4, kTurns = 8, kShareCtas = 2;
PartPlan part_plan(const Device *dev, int units, int nkv, int hd, long long rows, int tc) {
    PartPlan a;
    a.tc = tc > 0;
    a.rows = tc ? tc : kPtRows;
    a.row_tiles = (int)((rows + a.rows - 1) / a.rows);
    a.units = units * a.row_tiles;
    a.ctas = tc ? dev->sm_count : kShareCtas * dev->sm_count;
    const size_t items = (size_t)a.units * nkv;
    a.spans = (items * 8 + 15) / 16 * 16;
    a.most_chunks = items ? (int)std::max<size_t>(1, std::min<size_t>(kMostChunks, (size_t)kRounds * dev->sm_count / items)) : 1;
    a.slots = items == 0 ? 0 : ((size_t)a.ctas * 2 + items * (tc ? 1 : a.most_chunks)) * a.rows;
    a.bytes = a.slots * hd * 4 + a.slots * 8 + a.spans;
    return a;
}

struct PrefixPlan {
    PartPlan shared, own;
    size_t bytes;
};
// Shared rows that make CTAs for half of the places that the GPU has for them, in tiles of 16, are taken that way, whatever their number: a launch of paged_attn_tc.cu takes
// 18 us at least. (32 rows of a KV head behind 640, 80 CTAs: 18.5 us there, 12.3 here; behind 1500, 192: 21.6 and 14.6; 64 rows behind 1500, 384: 23.3 and 26.7.)
// bytes: enough for any max_prefix.
PrefixPlan prefix_plan(const Device *dev, const PagedView &v, int group, int max_new, int groups, int max_group_new, int max_prefix) {
    PrefixPlan a;
    const long long rows = (long long)max_group_new * group;
    const int tc = paged_tc_rows(v.hd, rows), chunk = v.hd == 256 ? 64 : 128;
    const PartPlan there = part_plan(dev, groups, v.nkv, v.hd, rows, tc), here = part_plan(dev, groups, v.nkv, v.hd, rows, 0);
    const bool few = (long long)here.units * v.nkv * ((max_prefix + (long long)chunk - 1) / chunk) <= 3ll * dev->sm_count / 2;
    a.shared = few ? here : there;
    a.own = part_plan(dev, v.nseq, v.nkv, v.hd, (long long)max_new * group, paged_tc_rows(v.hd, (long long)max_new * group));
    a.bytes = a.own.bytes + (tc && (long long)here.units * v.nkv <= 3ll * dev->sm_count / 2 ? std::max(here.bytes, there.bytes) : there.bytes);
    return a;
}

int prefix_check(const im_paged_kv *kv, int num_heads, int num_groups, int max_group_new) {
    IM_REQUIRE(num_groups >= 0 && max_group_new >= 1, "%d groups of %d new tokens", num_groups, max_group_new);
    const long long tiles = ((long long)(num_heads / kv->num_kv_heads) * max_group_new + 15) / 16;
    IM_REQUIRE(tiles <= (1 << 24) / std::max(num_groups, 1) / kv->num_kv_heads, "%d groups of %d new tokens are too many for one call", num_groups, max_group_new);
    return IM_OK;
}

// The launch's own: where its sums go, from `at` on.
unsigned char *lay_out(PartSet *s, const PartPlan &plan, int max_rows, int likely_rows, unsigned char *at) {
    PagedAttn *p = &s->p;
    s->rows = plan.rows;
    s->tc = plan.tc;
    p->row_tiles = plan.row_tiles;
    const long long items = (long long)plan.units * p->kv.nkv;
    const int chunk = p->kv.hd == 256 ? 64 : 128;
    p->ctas = (int)std::max(1ll, std::min<long long>(plan.ctas, items * ((max_rows + (plan.tc ? 128ll : chunk) - 1) / (plan.tc ? 128 : chunk))));
    s->chunks = plan.tc ? 1 : (int)std::max(1ll, std::min<long long>((likely_rows + (long long)chunk - 1) / chunk, plan.most_chunks));
    const bool long_ones = !plan.tc && items > 0 && (max_rows + (long long)chunk - 1) / chunk > (long long)s->chunks * kTurns;
    s->direct = long_ones ? s->chunks * kTurns : INT_MAX;
    s->share_ctas = long_ones ? p->ctas : 0;
    s->units = plan.units;
    s->cut_slot = plan.tc ? 0 : (int)(items * s->chunks);
    p->whole_slot = 2 * plan.ctas;
    p->part_o = reinterpret_cast<float *>(at);
    p->part_ml = reinterpret_cast<float2 *>(p->part_o + plan.slots * p->kv.hd);
    p->spans = reinterpret_cast<int *>(p->part_ml + plan.slots);
    p->odd = nullptr;  // (rows of parts are marked in part_ml)
    return at + plan.bytes;
}

template <bool BF16, int HD>
int part_launch(const Device *dev, const PrefixJoin &a, int shared_ctas, int own_ctas, cudaStream_t st) {
    using S = PtShape<HD>;
    static DeviceOnce once;
    if (once.first(dev->ordinal)) IM_CUDA_CHECK(cudaFuncSetAttribute((paged_part_kernel<BF16, HD>), cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    const int shares = (shared_ctas ? a.shared.share_ctas : 0) + (own_ctas ? a.own.share_ctas : 0);
    IM_CUDA_CHECK(launch_k(paged_part_kernel<BF16, HD>, dim3((unsigned)(shared_ctas + own_ctas + shares)), dim3(kPtThreads), (size_t)S::kSmem, st, a, shared_ctas, own_ctas));
    return IM_OK;
}

template <bool BF16, int HD>
int run(const Device *dev, PrefixJoin &a, const PrefixPlan &plan, cudaStream_t st) {
    const int nkv = a.own.p.kv.nkv;
    int rc = IM_OK, shared_ctas = 0, own_ctas = 0;
    if (plan.shared.units > 0) {
        if (plan.shared.tc) {
            a.shared.p.beside = !plan.own.tc;
            rc = paged_tc_part_launch(dev, a.shared.p, BF16, kShared, plan.shared.rows, plan.shared.units, st);
            a.own.p.early = 1;
        } else {
            shared_ctas = plan.shared.units * nkv * a.shared.chunks;
        }
    }
    if (rc != IM_OK) return rc;
    if (plan.own.tc) {
        if (shared_ctas) rc = part_launch<BF16, HD>(dev, a, shared_ctas, 0, st);
        if (rc == IM_OK) rc = paged_tc_part_launch(dev, a.own.p, BF16, kOwn, plan.own.rows, plan.own.units, st);
    } else {
        own_ctas = plan.own.units * nkv * a.own.chunks;
        rc = part_launch<BF16, HD>(dev, a, shared_ctas, own_ctas, st);
    }
    if (rc != IM_OK) return rc;
    const long long rows = (long long)a.own.p.tokens * a.own.p.group;
    IM_CUDA_CHECK(launch_k(paged_prefix_join_kernel<BF16, HD>, dim3((unsigned)((rows + kPjRows - 1) / kPjRows), (unsigned)nkv), dim3(2 * HD), 0, st, a));
    return IM_OK;
}

}  // namespace
}  // namespace im

IM_EXPORT size_t im_cuda_paged_prefix_attention_scratch_bytes(const im_device *dev, const im_paged_kv *kv, int num_heads, int max_new, int num_groups, int max_group_new) {
    try {
        im::PagedView v;
        if (!dev || im::paged_view(kv, 0, &v) != IM_OK || im::attn_check(kv, num_heads, max_new) != IM_OK || im::prefix_check(kv, num_heads, num_groups, max_group_new) != IM_OK) return 0;
        return im::prefix_plan(dev, v, num_heads / v.nkv, max_new, num_groups, max_group_new, 0).bytes;
    } catch (...) {
        return 0;
    }
}

IM_EXPORT int im_cuda_paged_prefix_attention(im_device *dev, const im_paged_kv *kv, const im_paged_prefix_args *args, void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    PrefixJoin a;
    PagedAttn &p = a.own.p;
    IM_REQUIRE(kv && args && kv->num_kv_heads > 0, "kv or args is NULL, or there are no heads");
    const im_paged_attention_args &x = args->attention;
    const int num_heads = x.num_heads, num_groups = args->num_groups, max_group_new = args->max_group_new;
    int rc = prefix_check(kv, num_heads, num_groups, max_group_new);
    if (rc != IM_OK) return rc;
    IM_REQUIRE(num_groups == 0 || (args->group_start_dev && args->prefix_pages_dev), "groups need their first sequences and numbers of shared pages");
    IM_REQUIRE(args->max_prefix >= 0, "max_prefix %d", args->max_prefix);
    bool empty;
    rc = attn_args(dev, kv, x.layer, x.q_dev, x.q_stride, x.out_dev, x.out_stride, num_heads, x.token_start_dev, x.num_tokens, x.max_new, x.mask_dev, x.mask_words, x.scale, x.max_len, &p, &empty);
    if (rc != IM_OK || empty) return rc;
    IM_REQUIRE(kv->num_kv_heads <= 65535, "at most 65535 key / value heads (got %d)", kv->num_kv_heads);
    const int max_len = attn_length(p.kv, x.max_len), max_prefix = std::min(attn_length(p.kv, args->max_prefix), max_len);
    const PrefixPlan plan = prefix_plan(dev, p.kv, p.group, x.max_new, num_groups, max_group_new, max_prefix);
    IM_REQUIRE(x.scratch_dev && aligned16(x.scratch_dev) && x.scratch_bytes >= plan.bytes, "paged prefix attention needs %zu bytes of 16-byte aligned scratch (got %zu)", plan.bytes,
               x.scratch_dev ? x.scratch_bytes : (size_t)0);
    p.group_start = args->group_start_dev;
    p.prefix_pages = args->prefix_pages_dev;
    p.groups = num_groups;
    a.shared.p = p;
    a.shared.p.mask = nullptr;
    a.shared.p.max_new = max_group_new;
    a.group_new = max_group_new;
    unsigned char *at = lay_out(&a.shared, plan.shared, plan.shared.tc ? max_prefix : max_len, max_prefix, static_cast<unsigned char *>(x.scratch_dev));
    lay_out(&a.own, plan.own, max_len, num_groups ? std::max(1, max_len - max_prefix) : max_len, at);
    const cudaStream_t st = as_stream(stream);
    const bool bf16 = kv->dtype == IM_DTYPE_BF16;
#define IM_RUN(HD) (bf16 ? run<true, HD>(dev, a, plan, st) : run<false, HD>(dev, a, plan, st))
    switch (kv->head_dim) {
    case 64: return IM_RUN(64);
    case 128: return IM_RUN(128);
    default: return IM_RUN(256);
    }
#undef IM_RUN
    IM_GUARD_END
}
