// Attention of new tokens (one of each sequence, a portion of a prompt, or a tree of drafted tokens) over a paged cache.
//
//   out[t, h] = sum_j p_j v_j,  p = softmax over the visible rows j of scale * q[t, h] . k_j
//
// What bounds it is the read of K and V: every (sequence, KV head) is read once for all the rows (token, query head) that share it, here up
// to 16 (more: paged_attn_tc.cu). 32 sequences of up to 8192 rows, 32 / 8 heads (579 MB): 106 us, 5.5 TB/s, 84 % of a copy. The tiles of 64 positions of all (row tile, KV head) items form one list, cut into equal shares, one per CTA, whatever the lengths
// are; an item that a cut divides leaves partial sums, which a second launch joins.
//
// In a CTA four warps take 16 positions of each tile and work on their own: each keeps a ring of K and V slices (cp.async, 16 bytes per lane, rows
// looked up in the page table, so that any page size works and pages may end anywhere) and its own running maximum, sum and outputs of all
// rows; they meet only where an item ends. The ring runs ahead over the ends of items. Scores and outputs on mma.sync m16n8k16 (a
// tile of 64 positions against 16 rows is 256 instructions for 32 KB: far from what bounds it), weights as two 16-bit terms.
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "cluster.cuh"
#include "paged_attn.cuh"

namespace im {
namespace {

constexpr int kPaWarps = 4, kPaThreads = kPaWarps * 32, kPaSlice = 16, kPaTile = kPaWarps * kPaSlice;

template <int HD>
struct PaShape {
    static constexpr int kRows = 16;
    static constexpr int kSliceBytes = kPaSlice * HD * 2;
    static constexpr int kStages = HD == 64 ? 6 : 3;
    static constexpr int kRing = kPaWarps * kStages * 2 * kSliceBytes;
    static constexpr int kMerge = kRows * HD * 4;
    static constexpr int kSmem = kRing + kMerge + kPaWarps * kRows * 8;
};

// CL: instead of shares of the list of all tiles, a cluster of CTAs per item, each with an equal run of its tiles; they join what they have
// through each other's shared memory, in the same launch and without scratch.
template <bool BF16, int HD, bool CL, int MODE>
__global__ void __launch_bounds__(kPaThreads, HD == 256 ? 1 : 2) paged_attn_kernel(const __grid_constant__ PagedAttn p, int units) {
    using S = PaShape<HD>;
    // fp16 weights: 2^15 at the row's maximum instead of 1, so that they are normal numbers down to 2^-29 of it (exact to 2^-40 below)
    constexpr float kLift = BF16 ? 0.0f : 15.0f;
    constexpr int R = S::kRows, KS = HD / 16, NT = HD / 8, CH = HD / 8;  // k steps, 8-column tiles, 16-byte pieces of a row
    extern __shared__ __align__(128) unsigned char pa_smem[];
    __shared__ long long sums[kPaThreads + kShareMore];
    __shared__ unsigned rows_there[kPaWarps][8];  // of a slice in the ring: bit r where row r is in the cache
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned char *ring = pa_smem + warp * (S::kRing / kPaWarps);
    float *merge = reinterpret_cast<float *>(pa_smem + S::kRing);
    float2 *ml = reinterpret_cast<float2 *>(reinterpret_cast<unsigned char *>(merge) + S::kMerge);  // [warps, R]
    __shared__ unsigned bad_rows[2];  // rows of an item whose sums are not finite, every other item's
    __shared__ float2 joint[CL ? R : 1];  // maximum and sum of this CTA's part of each row
    if (tid < 2) bad_rows[tid] = 0;
    pdl_trigger();
    pdl_wait();
    Share share;
    PagedUnit f_u;  // the unit that the copies are at
    if constexpr (CL) {
        const int C = (int)cluster_size(), item = blockIdx.x / C, rank = (int)cluster_rank();
        share.unit = item / p.kv.nkv;
        share.head = item - share.unit * p.kv.nkv;
        f_u = paged_unit<R, MODE>(p, share.unit);
        const int n = unit_tiles<kPaTile, MODE>(f_u);
        if (n == 0) return;  // all of the cluster
        share.from = share.tile = (int)((long long)n * rank / C);
        share.to = (long long)n * (rank + 1) / C;
    } else {
        share = units <= 32 ? warp_share<R, kPaTile, MODE>(p, units, p.ctas, f_u) : find_share<R, kPaTile, kPaThreads, MODE>(p, units, p.ctas, sums, f_u);
        if (share.from >= share.to) return;
    }
    const int count = (int)(share.to - share.from);

    // ---- the copies' cursor: one slice ahead of the copies, so that a page number is there when it is needed
    int f_unit = share.unit, f_head = share.head, f_tile = share.tile, f_left = count;
    int f_tiles = unit_tiles<kPaTile, MODE>(f_u);
    int n_page = -1, n_slot = 0, n_head = 0;  // of the slice that is copied next: this lane's row (lane & 15)
    auto fetch = [&]() {
        n_page = -1;
        if (f_left <= 0) return;
        const int pos = f_tile * kPaTile + warp * kPaSlice + (lane & 15);
        if (pos < f_u.end) {
            const int pg = pos / p.kv.page;
            n_slot = pos - pg * p.kv.page;
            n_page = __ldg(p.kv.table + f_u.seq * p.kv.table_stride + pg);
        }
        n_head = f_head;
        f_left--;
        if (++f_tile == f_tiles) {
            f_tile = 0;
            if (++f_head == p.kv.nkv) {
                f_head = 0;
                while (f_left > 0 && ++f_unit < units) {
                    f_u = paged_unit<R, MODE>(p, f_unit);
                    f_tiles = unit_tiles<kPaTile, MODE>(f_u);
                    if (f_tiles > 0) break;
                }
            }
        }
    };
    auto copy = [&](int stage) {  // the slice whose rows fetch() looked up
        const bool there = (unsigned)n_page < (unsigned)p.kv.pages;
        const long long off = there ? n_page * p.kv.page_stride + ((long long)n_head * p.kv.page + n_slot) * HD : -1;
        const uint32_t dst = smem_u32(ring) + stage * 2 * S::kSliceBytes;
        const unsigned all = __ballot_sync(0xffffffffu, there);
        if (lane == 0) rows_there[warp][stage] = all;
        constexpr int RPI = 32 / CH > 0 ? 32 / CH : 1;  // rows of one request of the warp
        constexpr int IPR = CH / 32 > 0 ? CH / 32 : 1;
#pragma unroll
        for (int i = 0; i < kPaSlice / RPI; i++) {
            const int row = i * RPI + (RPI > 1 ? lane / CH : 0);
            const long long at = __shfl_sync(0xffffffffu, off, row);
#pragma unroll
            for (int j = 0; j < IPR; j++) {
                const int c = (lane & (CH < 32 ? CH - 1 : 31)) + j * 32;
                const uint32_t d = dst + row * (HD * 2) + ((c ^ (row & 7)) << 4);
                const long long src = at < 0 ? 0 : at + c * 8;
                cp16(d, p.kc + src, at >= 0);
                cp16(d + S::kSliceBytes, p.vc + src, at >= 0);
            }
        }
    };
    fetch();
#pragma unroll
    for (int i = 0; i < S::kStages - 1; i++) {
        if (i < count) {
            copy(i);
            fetch();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // ---- the items
    int unit = share.unit, head = share.head, tile = share.tile, done = 0, stage = 0;
    bool first_item = true;
    int odd_item = 0;
    while (done < count) {
        PagedUnit u = paged_unit<R, MODE>(p, unit);
        const int tiles = unit_tiles<kPaTile, MODE>(u);
        if (tiles == 0) {
            unit++;
            continue;
        }
        const int t0 = tile, t1 = min(tiles, tile + count - done);
        // queries: A fragments, rows lane / 4 and lane / 4 + 8 of each 16
        uint32_t qf[KS][4];
        int tok[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = (lane >> 2) + 8 * i;
            tok[i] = (u.row0 + min(r, u.rows - 1)) / p.group;
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = (lane >> 2) + 8 * i;
            const uint32_t *src = reinterpret_cast<const uint32_t *>(p.q + (u.tok0 + tok[i]) * p.qs + (long long)(head * p.group + (u.row0 + r) % p.group) * HD);
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int j = 0; j < 2; j++) qf[ks][2 * j + i] = r < u.rows ? __ldg(src + ks * 8 + j * 4 + (lane & 3)) : 0u;
        }
        float m[2], l[2], o[NT][4];
#pragma unroll
        for (int i = 0; i < 2; i++) m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[n][j] = 0.0f;
        for (; tile < t1; tile++, done++) {
            // the next slice on its way, this one there
            if (done + S::kStages - 1 < count) {
                int to = stage + S::kStages - 1;
                if (to >= S::kStages) to -= S::kStages;
                copy(to);
                fetch();
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
            __syncwarp();
            const uint32_t ks_at = smem_u32(ring) + stage * 2 * S::kSliceBytes, vs_at = ks_at + S::kSliceBytes;
            float s[2][4];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[n][j] = 0.0f;
            {
                const int r = (lane & 7) + ((lane >> 4) << 3), hi = (lane >> 3) & 1;  // row and 16-byte half of this lane's matrix row
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uint32_t b[4];
                    ldsm4(b, ks_at + r * (HD * 2) + (((2 * ks + hi) ^ (r & 7)) << 4));
                    mma16<BF16>(s[0], qf[ks], b[0], b[1]);
                    mma16<BF16>(s[1], qf[ks], b[2], b[3]);
                }
            }
            const int pos0 = tile * kPaTile + warp * kPaSlice;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[n][j] *= p.scale2;
            const unsigned there = rows_there[warp][stage] & 0xffffu;
            if (there != 0xffffu || pos0 + kPaSlice > u.len) {  // some row may not see some position
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int at = n * 8 + (lane & 3) * 2 + (j & 1);
                        if (!(there >> at & 1) || !paged_sees(p, u, tok[j >> 1], pos0 + at)) s[n][j] = -INFINITY;
                    }
            }
            if (MODE == kWeigh && p.scores && pos0 < p.score_cap) {  // (a multiple of a tile)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int r = (lane >> 2) + 8 * i;
                    float *to = p.scores + (((long long)unit * p.kv.nkv + head) * p.score_rows + r) * p.score_cap + pos0 + (lane & 3) * 2;
                    if (r < u.rows)
#pragma unroll
                        for (int n = 0; n < 2; n++) *reinterpret_cast<float2 *>(to + n * 8) = make_float2(s[n][2 * i], s[n][2 * i + 1]);
                }
            }
            uint32_t w[4], w2[4];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float top = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                if (__any_sync(0xffffffffu, top > m[i])) {
                    const float m_new = fmaxf(m[i], top), corr = m_new == -INFINITY ? 1.0f : ex2(m[i] - m_new);
                    m[i] = m_new;
                    l[i] *= corr;
#pragma unroll
                    for (int n = 0; n < NT; n++) o[n][2 * i] *= corr, o[n][2 * i + 1] *= corr;
                }
                const float base = m[i] == -INFINITY ? 0.0f : m[i] - kLift;
                float sum = 0.0f;
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const float x0 = ex2(s[n][2 * i] - base), x1 = ex2(s[n][2 * i + 1] - base);
                    sum += x0 + x1;
                    w[2 * n + i] = pack16<BF16>(x0, x1);
                    const float2 back = unpack16<BF16>(w[2 * n + i]);
                    w2[2 * n + i] = pack16<BF16>(x0 - back.x, x1 - back.y);
                }
                l[i] += sum;
            }
            {
                const int r = (lane & 7) + (((lane >> 3) & 1) << 3), hi = lane >> 4;
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t b[4];
                    ldsm4t(b, vs_at + r * (HD * 2) + (((n + hi) ^ (r & 7)) << 4));
                    mma16<BF16>(o[n], w, b[0], b[1]);
                    mma16<BF16>(o[n + 1], w, b[2], b[3]);
                    mma16<BF16>(o[n], w2, b[0], b[1]);
                    mma16<BF16>(o[n + 1], w2, b[2], b[3]);
                }
            }
            __syncwarp();  // every lane has read the slice before the copies of the one that takes its place
            if (++stage == S::kStages) stage = 0;
        }
        // ---- the item's (or the share's part of it) rows: four warps' sums joined in order
#pragma unroll
        for (int i = 0; i < 2; i++) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if ((lane & 3) == 0) ml[warp * R + (lane >> 2) + 8 * i] = make_float2(m[i], l[i]);
        }
        __syncthreads();
        if (tid == 0) bad_rows[!odd_item] = 0;  // every thread has looked at the last item's
        const bool whole = !CL && t0 == 0 && t1 == tiles;
        const size_t part = ((size_t)blockIdx.x * 2 + (first_item ? 0 : 1)) * R;
        if (!CL && tid == 0) note_span<MODE>(p, unit, head, t0, t1, tiles, blockIdx.x, first_item ? 0 : 1);
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = (lane >> 2) + 8 * i;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kPaWarps; w++) M = fmaxf(M, ml[w * R + r].x);
            f[i] = m[i] == -INFINITY && l[i] == 0.0f ? 0.0f : ex2(m[i] - M);
        }
        auto row_ml = [&](int r) {
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < kPaWarps; w++) M = fmaxf(M, ml[w * R + r].x);
#pragma unroll
            for (int w = 0; w < kPaWarps; w++) {
                const float2 x = ml[w * R + r];
                L += x.x == -INFINITY && x.y == 0.0f ? 0.0f : x.y * ex2(x.x - M);
            }
            return make_float2(M - kLift, L);  // (plain_row has no lift)
        };
#pragma unroll 1
        for (int w = 0; w < kPaWarps; w++) {
            if (warp == w) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        float2 *at = reinterpret_cast<float2 *>(merge + ((lane >> 2) + 8 * i) * HD + ((n * 8 + (lane & 3) * 2) ^ (((lane >> 2) & 3) << 3)));
                        float2 x = make_float2(o[n][2 * i] * f[i], o[n][2 * i + 1] * f[i]);
                        if (f[i] == 0.0f) x = make_float2(0.0f, 0.0f);
                        if (w > 0) {
                            const float2 y = *at;
                            x.x += y.x;
                            x.y += y.y;
                        }
                        *at = x;
                    }
            }
            __syncthreads();
        }
        for (int i = tid; i < u.rows * CH; i += kPaThreads) {
            const int r = i / CH, c = i % CH * 8;
            const float *src = merge + r * HD + (c ^ ((r & 3) << 3));
            float v[8], worst = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j += 4) *reinterpret_cast<float4 *>(v + j) = *reinterpret_cast<const float4 *>(src + j);
#pragma unroll
            for (int j = 0; j < 8; j++) worst += v[j] * 0.0f;  // zero unless a value is not finite
            if (worst != 0.0f) atomicOr(&bad_rows[odd_item], 1u << r);
            if (whole) {
                const float2 x = row_ml(r);
                const float inv = x.y > 0.0f ? 1.0f / x.y : x.y == 0.0f ? 0.0f : x.y;
                const int t = (u.row0 + r) / p.group, g = (u.row0 + r) % p.group;
                *reinterpret_cast<uint4 *>(p.out + (u.tok0 + t) * p.os + (long long)(head * p.group + g) * HD + c) =
                    make_uint4(pack16<BF16>(v[0] * inv, v[1] * inv), pack16<BF16>(v[2] * inv, v[3] * inv), pack16<BF16>(v[4] * inv, v[5] * inv),
                               pack16<BF16>(v[6] * inv, v[7] * inv));
            } else if (!CL) {
                float4 *dst = reinterpret_cast<float4 *>(p.part_o + (part + r) * HD + c);
                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                dst[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
        if (!whole)
            for (int r = tid; r < u.rows; r += kPaThreads) {
                if (CL) joint[r] = row_ml(r);
                else p.part_ml[part + r] = row_ml(r);
            }
        if (MODE == kWeigh && whole)
            for (int r = tid; r < u.rows; r += kPaThreads) p.stat[((long long)unit * p.kv.nkv + head) * R + r] = row_ml(r);
        __syncthreads();
        if (const unsigned bad = bad_rows[odd_item]) {
            for (int r = warp; r < u.rows; r += kPaWarps) {
                if (!(bad >> r & 1)) continue;
                float x[HD / 32], M, L;
                plain_row<BF16, HD>(p, u, head, r, t0 * kPaTile, min(t1 * kPaTile, u.end), x, M, L);
                const int t = (u.row0 + r) / p.group, g = (u.row0 + r) % p.group;
                const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
                for (int i = 0; i < HD / 32; i++) {
                    if (whole) p.out[(u.tok0 + t) * p.os + (long long)(head * p.group + g) * HD + lane + 32 * i] = (uint16_t)pack16<BF16>(x[i] * inv, 0.0f);
                    else if (CL) merge[r * HD + ((lane + 32 * i) ^ ((r & 3) << 3))] = x[i];
                    else p.part_o[(part + r) * HD + lane + 32 * i] = x[i];
                }
                if (!whole && lane == 0) (CL ? joint[r] : p.part_ml[part + r]) = make_float2(M, L);
            }
            __syncthreads();
        }
        first_item = false;
        odd_item ^= 1;
        if (t1 == tiles) {
            tile = 0;
            if (++head == p.kv.nkv) {
                head = 0;
                unit++;
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if constexpr (CL) {
        const int C = (int)cluster_size(), rank = (int)cluster_rank();
        if (count == 0 && tid < R) joint[tid] = make_float2(-INFINITY, 0.0f);
        cluster_sync();
        const PagedUnit u = paged_unit<R, MODE>(p, share.unit);
        for (int i = rank * kPaThreads + tid; i < u.rows * CH; i += C * kPaThreads) {
            const int r = i / CH, c = i % CH * 8;
            float M = -INFINITY, L = 0.0f, o[8];
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] = 0.0f;
            for (int k = 0; k < C; k++) M = fmaxf(M, remote2(of_rank(joint + r, k)).x);
#pragma unroll 1
            for (int k = 0; k < C; k++) {
                const float2 x = remote2(of_rank(joint + r, k));
                if (x.x == -INFINITY && x.y == 0.0f) continue;  // nothing seen in this part
                const uint32_t at = of_rank(merge + r * HD + (c ^ ((r & 3) << 3)), k);
                const float4 a = remote4(at), b = remote4(at + 16);
                const float f = ex2(x.x - M);
                L += x.y * f;
                o[0] += a.x * f; o[1] += a.y * f; o[2] += a.z * f; o[3] += a.w * f;
                o[4] += b.x * f; o[5] += b.y * f; o[6] += b.z * f; o[7] += b.w * f;
            }
            const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
            const int t = (u.row0 + r) / p.group, g = (u.row0 + r) % p.group;
            *reinterpret_cast<uint4 *>(p.out + (u.tok0 + t) * p.os + (long long)(share.head * p.group + g) * HD + c) =
                make_uint4(pack16<BF16>(o[0] * inv, o[1] * inv), pack16<BF16>(o[2] * inv, o[3] * inv), pack16<BF16>(o[4] * inv, o[5] * inv), pack16<BF16>(o[6] * inv, o[7] * inv));
        }
        if constexpr (MODE == kWeigh) {  // the sums of this CTA's positions
            __shared__ float norms[R];
            if (tid < u.rows) {
                float M = -INFINITY, L = 0.0f;
                for (int k = 0; k < C; k++) M = fmaxf(M, remote2(of_rank(joint + tid, k)).x);
                for (int k = 0; k < C; k++) {
                    const float2 x = remote2(of_rank(joint + tid, k));
                    if (!(x.x == -INFINITY && x.y == 0.0f)) L += x.y * ex2(x.x - M);
                }
                norms[tid] = row_norm(make_float2(M, L));
                if (!p.scores && rank == 0) p.stat[(long long)(blockIdx.x / C) * R + tid] = make_float2(M, L);
            }
            __syncthreads();
            const float *scores = p.scores + (long long)(blockIdx.x / C) * p.score_rows * p.score_cap;
            for (int pos = (int)share.from * kPaTile + tid; p.scores && pos < min((int)share.to * kPaTile, u.end); pos += kPaThreads) {
                float v = 0.0f;
                if (pos >= p.score_cap) v = plain_sum<BF16, HD>(p, u, share.head, pos, norms);
                else
                    for (int r = 0; r < u.rows; r++) v += ex2(scores[(long long)r * p.score_cap + pos] + norms[r]);
                add_sum(p, u, share.head, pos, seen_sum<BF16, HD>(p, u, share.head, pos, norms, v));
            }
        }
        cluster_sync();  // nobody leaves while another reads what it has
    }
}

// Items that a cut divides: eight rows a block.
constexpr int kJoinWarps = 8;
template <bool BF16, int R, int HD>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const __grid_constant__ PagedAttn p) {
    pdl_trigger();
    pdl_wait();
    join_row<BF16, R, HD>(p, blockIdx.x, blockIdx.y * kJoinWarps + (threadIdx.x >> 5));
}


constexpr int kClusterMost = 8;

}  // namespace

AttnPlan attn_plan(const Device *dev, int nseq, int nkv, int hd, int group, int max_new, int max_len) {
    AttnPlan a;
    // Up to 16 rows of a KV head (and heads of 256, whose scores and outputs tensor memory does not hold twice) on mma.sync, more on tcgen05. Eight sequences of
    // up to 4001 rows: 16 rows 29.7 us here, 28.6 there; 8 rows 27.6 and 28.5; 20 rows as two tiles of 16: 40 and 29. 32 sequences of up to 8192, one token
    // each (4 rows): 103 and 122.
    const int tc = paged_tc_rows(hd, (long long)group * max_new);
    a.tile = tc ? 128 : kPaTile;
    a.rows = tc ? tc : 16;
    a.row_tiles = (int)(((long long)group * max_new + a.rows - 1) / a.rows);
    a.units = nseq * a.row_tiles;
    a.ctas = dev->sm_count * (tc || hd == 256 ? 1 : 2);
    // Contexts that the GPU's CTAs, as many for every item, read in up to 16 tiles each (8 where an item has eight CTAs and not all of the GPU's are used): a cluster
    // per item, one launch. 32 sequences of up to 1000 rows 25 us, 33 in shares; of 2000 (32 tiles) 42 and 43, of 8192 140 and 102; one of 4000 (8 tiles for
    // each of eight CTAs) 16.8 and 17.2, of 8000 24 and 20.
    const long long items = (long long)a.units * nkv, tiles = (max_len + (long long)kPaTile - 1) / kPaTile;
    a.cluster = (int)std::max(1ll, std::min({(long long)a.ctas / std::max(items, 1ll), tiles, (long long)kClusterMost}));
    if (a.rows != 16 || tiles > (a.cluster < kClusterMost ? 16ll : 8ll) * a.cluster) a.cluster = 0;
    if (a.cluster) {
        a.bytes = 0;
        return a;
    }
    const size_t slots = (size_t)a.ctas * 2 * a.rows;
    a.bytes = slots * hd * 4 + slots * 8 + (size_t)items * (tc ? 40 : 8);
    return a;
}

void attn_lay_out(PagedAttn *p, const AttnPlan &plan, int max_len, void *at) {
    p->row_tiles = plan.row_tiles;
    // no more CTAs than tiles
    const long long tiles = (long long)plan.units * p->kv.nkv * ((max_len + (long long)plan.tile - 1) / plan.tile);
    p->ctas = (int)std::max(1ll, std::min<long long>(plan.ctas, tiles));
    const size_t slots = (size_t)plan.ctas * 2 * plan.rows;
    p->part_o = static_cast<float *>(at);
    p->part_ml = reinterpret_cast<float2 *>(p->part_o + slots * p->kv.hd);
    p->spans = reinterpret_cast<int *>(p->part_ml + slots);
    p->odd = reinterpret_cast<unsigned *>(p->spans + 2ll * plan.units * p->kv.nkv);
}

namespace {

template <bool BF16, int R, int HD>
int join_launch(const PagedAttn &p, int units, cudaStream_t st) {
    const long long rows = std::min<long long>(R, (long long)p.max_new * p.group);
    IM_CUDA_CHECK(launch_k(paged_join_kernel<BF16, R, HD>, dim3((unsigned)(units * p.kv.nkv), (unsigned)((rows + kJoinWarps - 1) / kJoinWarps)), dim3(kJoinWarps * 32), 0, st, p));
    return IM_OK;
}

template <bool BF16, int HD, int MODE>
int attn_launch(const Device *dev, const PagedAttn &p, int units, int cluster, bool joins, cudaStream_t st) {
    using S = PaShape<HD>;
    static DeviceOnce once;
    if (once.first(dev->ordinal)) {
        IM_CUDA_CHECK(cudaFuncSetAttribute((paged_attn_kernel<BF16, HD, false, MODE>), cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
        IM_CUDA_CHECK(cudaFuncSetAttribute((paged_attn_kernel<BF16, HD, true, MODE>), cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    }
    if (cluster) {
        IM_CUDA_CHECK(launch_cluster(paged_attn_kernel<BF16, HD, true, MODE>, dim3((unsigned)(units * p.kv.nkv * cluster)), dim3(kPaThreads), cluster, (size_t)S::kSmem, st, p, units));
        return IM_OK;
    }
    IM_CUDA_CHECK(launch_k(paged_attn_kernel<BF16, HD, false, MODE>, dim3(p.ctas), dim3(kPaThreads), (size_t)S::kSmem, st, p, units));
    return joins ? join_launch<BF16, S::kRows, HD>(p, units, st) : IM_OK;
}

}  // namespace

int paged_weigh_launch(const Device *dev, const PagedAttn &p, bool bf16, int units, int cluster, bool joins, cudaStream_t st) {
#define IM_RUN(HD) (bf16 ? attn_launch<true, HD, kWeigh>(dev, p, units, cluster, joins, st) : attn_launch<false, HD, kWeigh>(dev, p, units, cluster, joins, st))
    switch (p.kv.hd) {
    case 64: return IM_RUN(64);
    case 128: return IM_RUN(128);
    default: return IM_RUN(256);
    }
#undef IM_RUN
}

// Rows that no sequence passes.
int attn_length(const PagedView &v, int max_len) { return max_len > 0 && max_len < v.rows ? max_len : v.rows; }

int attn_check(const im_paged_kv *kv, int num_heads, int max_new) {
    IM_REQUIRE(kv->head_dim == 64 || kv->head_dim == 128 || kv->head_dim == 256, "paged attention is built for heads of 64, 128 and 256 (got %d)", kv->head_dim);
    IM_REQUIRE(num_heads > 0 && num_heads % kv->num_kv_heads == 0, "num_heads has to be a multiple of num_kv_heads (got %d and %d)", num_heads, kv->num_kv_heads);
    IM_REQUIRE(max_new >= 1, "max_new has to be at least 1 (got %d)", max_new);
    const long long tiles = ((long long)(num_heads / kv->num_kv_heads) * max_new + 15) / 16;
    IM_REQUIRE(tiles <= (1 << 24) / std::max(kv->num_seqs, 1) / kv->num_kv_heads, "%d sequences of %d new tokens are too many for one call", kv->num_seqs, max_new);
    return IM_OK;
}

// What calls have in common: their arguments checked, p filled in but for the plan. empty: there is nothing to do.
int attn_args(im_device *dev, const im_paged_kv *kv, int layer, const void *q_dev, int64_t q_stride, void *out_dev, int64_t out_stride, int num_heads,
              const int *token_start_dev, int num_tokens, int max_new, const uint64_t *mask_dev, int mask_words, float scale, int max_len, PagedAttn *p, bool *empty) {
    *empty = false;
    IM_REQUIRE(layer >= 0, "layer %d", layer);
    int rc = paged_view(kv, layer, &p->kv);
    if (rc == IM_OK) rc = attn_check(kv, num_heads, max_new);
    if (rc != IM_OK) return rc;
    IM_REQUIRE(num_tokens >= 0 && max_len >= 0, "bad argument");
    if (num_tokens == 0 || kv->num_seqs == 0) {
        *empty = true;
        return paged_device(dev);
    }
    IM_REQUIRE(q_dev && out_dev && token_start_dev, "bad argument");
    const int64_t row = (int64_t)num_heads * kv->head_dim, most = (int64_t)1 << 40;
    IM_REQUIRE(q_stride >= row && out_stride >= row && q_stride <= most && out_stride <= most && q_stride % 8 == 0 && out_stride % 8 == 0 && aligned16(q_dev) && aligned16(out_dev),
               "rows of queries and outputs have to be 16-byte aligned and apart");
    IM_REQUIRE(!share_rows(q_dev, 2 * q_stride, out_dev, 2 * out_stride, 2 * row, num_tokens), "the outputs lie over the queries");
    IM_REQUIRE(!mask_dev || (mask_words >= 1 && mask_words <= 1 << 20), "a mask of %d words a token", mask_words);
    IM_REQUIRE(scale == scale && scale - scale == 0.0f, "scale is not finite");
    rc = paged_device(dev);
    if (rc != IM_OK) return rc;
    const int64_t at = layer * (int64_t)p->kv.layer_stride;
    p->kc = static_cast<const uint16_t *>(kv->k_dev) + at;
    p->vc = static_cast<const uint16_t *>(kv->v_dev) + at;
    p->q = static_cast<const uint16_t *>(q_dev);
    p->out = static_cast<uint16_t *>(out_dev);
    p->qs = q_stride; p->os = out_stride;
    p->start = token_start_dev;
    p->mask = mask_dev; p->mask_words = mask_words;
    p->group = num_heads / kv->num_kv_heads; p->tokens = num_tokens; p->max_new = max_new;
    p->scale2 = scale * 1.4426950408889634f;
    if (p->scale2 == 0.0f) p->scale2 = 1e-30f;  // every position alike, without 0 * inf at the hidden ones
    p->group_start = p->prefix_pages = nullptr;
    p->groups = p->whole_slot = p->beside = p->early = 0;
    p->stat = p->stat_parts = nullptr;
    p->scores = p->sums = nullptr;
    return IM_OK;
}

}  // namespace im

IM_EXPORT size_t im_cuda_paged_attention_scratch_bytes(const im_device *dev, const im_paged_kv *kv, int num_heads, int max_new, int max_len) {
    try {
        im::PagedView v;
        if (!dev || im::paged_view(kv, 0, &v) != IM_OK || im::attn_check(kv, num_heads, max_new) != IM_OK) return 0;
        if (max_len < 0) return 0;
        return im::attn_plan(dev, v.nseq, v.nkv, v.hd, num_heads / v.nkv, max_new, im::attn_length(v, max_len)).bytes;
    } catch (...) {
        return 0;
    }
}

IM_EXPORT int im_cuda_paged_attention(im_device *dev, const im_paged_kv *kv, int layer, const void *q_dev, int64_t q_stride, void *out_dev, int64_t out_stride,
                                      int num_heads, const int *token_start_dev, int num_tokens, int max_new, const uint64_t *mask_dev, int mask_words,
                                      float scale, int max_len, void *scratch_dev, size_t scratch_bytes, void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    PagedAttn p;
    bool empty;
    const int rc = attn_args(dev, kv, layer, q_dev, q_stride, out_dev, out_stride, num_heads, token_start_dev, num_tokens, max_new, mask_dev, mask_words, scale, max_len, &p, &empty);
    if (rc != IM_OK || empty) return rc;
    max_len = attn_length(p.kv, max_len);
    const AttnPlan plan = attn_plan(dev, p.kv.nseq, p.kv.nkv, p.kv.hd, num_heads / kv->num_kv_heads, max_new, max_len);
    IM_REQUIRE(plan.bytes == 0 || (scratch_dev && aligned16(scratch_dev) && scratch_bytes >= plan.bytes), "paged attention needs %zu bytes of 16-byte aligned scratch (got %zu)", plan.bytes,
               scratch_dev ? scratch_bytes : (size_t)0);
    attn_lay_out(&p, plan, max_len, scratch_dev);
    const cudaStream_t st = as_stream(stream);
    const bool bf16 = kv->dtype == IM_DTYPE_BF16;
    if (plan.rows >= 128) return paged_tc_launch(dev, p, bf16, plan.rows, plan.units, st);
#define IM_RUN(HD) (bf16 ? attn_launch<true, HD, kAttend>(dev, p, plan.units, plan.cluster, true, st) : attn_launch<false, HD, kAttend>(dev, p, plan.units, plan.cluster, true, st))
    switch (kv->head_dim) {
    case 64: return IM_RUN(64);
    case 128: return IM_RUN(128);
    default: return IM_RUN(256);
    }
#undef IM_RUN
    IM_GUARD_END
}
