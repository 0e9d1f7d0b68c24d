// Attention over a paged cache: what its kernels share (paged_attn.cu).
#pragma once
#include "paged.cuh"
#include "umma.cuh"

namespace im {

struct PagedAttn {
    PagedView kv;
    const uint16_t *kc, *vc;  // of the layer
    const uint16_t *q;
    uint16_t *out;
    long long qs, os;
    const int *start;
    const uint64_t *mask;
    int mask_words, group, tokens, max_new;
    float scale2;             // scale / ln 2: scores in powers of two
    int row_tiles;            // row tiles of a sequence: ceil(max_new * group / rows of a tile)
    int ctas;                 // CTAs of the attention kernel
    float *part_o;            // [ctas, 2, rows of a tile, head_dim]: sums of weighted values
    float2 *part_ml;          // [ctas, 2, rows of a tile]: maximum, sum of weights
    int *spans;               // [units, KV heads, 2]: the slot of an item's first part (-1: one CTA had all of it), the CTA of its last one
    unsigned *odd;            // tcgen05: [units, KV heads, 8]: rows of an item that one CTA had whose sums are not finite (rows of parts: a NaN in part_ml)
    // sequences in groups that share their first pages (paged_prefix.cu)
    const int *group_start, *prefix_pages;  // [groups + 1] sequences, [groups]
    int groups;
    int whole_slot;           // kShared, kOwn: slots from here on are those of items that one CTA had, by item
    int beside;               // kShared: the own rows are read by others at the same time, only as many CTAs as shared_ctas_beside() says take part
    int early;                // kOwn: a kShared launch that this one needs nothing of may still run (see paged_prefix.cu)
    // sums of softmax weights (paged_weights.cu)
    float2 *stat;             // [units, KV heads, rows of a tile]: maximum and sum of weights of every row of an item that one CTA (or cluster) had
    float2 *stat_parts;       // tcgen05: [slots, rows of a tile]: of the others' parts, where part_ml may have a NaN instead
    float *scores;            // or NULL: [units, KV heads, score_rows, score_cap]: scores of the positions before score_cap, in powers of two
    int score_cap, score_rows;
    float *sums;              // [sequences, KV heads, sum_cols]
    long long sum_seq, sum_head;
    int sum_cols;
};

// What a launch computes: attention; the part of it over the pages that a group of sequences shares, all the group's rows together; the part over the
// rows of their own. The parts leave sums (never outputs) for another launch to join. kWeigh: attention that says what each row's weights were normed by, and
// where there is room for them the scores.
enum PagedMode { kAttend, kShared, kOwn, kWeigh };
template <int MODE>
constexpr bool whole_items() { return MODE == kAttend || MODE == kWeigh; }  // an item that one CTA had is done

// A unit: a tile of rows (token, query head of the KV head) of one sequence, rows token-major.
struct PagedUnit {
    int seq, row0, rows;      // first row among the sequence's; rows of it that exist
    int tok0;                 // the sequence's first new token
    int len, fresh;           // rows before the new ones; new ones that lie in the table
    int end;                  // no row of the unit sees a position from here on
    int from;                 // kOwn: its first position
};
template <int MODE>
__device__ __forceinline__ int unit_from(const PagedUnit &u) { return MODE == kOwn ? u.from : 0; }

// The group of a sequence, -1 where it has none: the last that starts at or before it.
__device__ __forceinline__ int paged_group_of(const PagedAttn &p, int seq) {
    if (p.groups == 0 || seq < __ldg(p.group_start) || seq >= __ldg(p.group_start + p.groups)) return -1;
    int lo = 0, hi = p.groups;  // it lies in [lo, hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (__ldg(p.group_start + mid) <= seq) lo = mid;
        else hi = mid;
    }
    return lo;
}
// Rows that the sequences of a group share.
__device__ __forceinline__ int prefix_rows(const PagedAttn &p, int group) { return group < 0 ? 0 : min(max(__ldg(p.prefix_pages + group), 0), p.kv.width) * p.kv.page; }

template <int MODE>
__device__ __forceinline__ PagedUnit paged_unit_of(const PagedAttn &p, int u, int R) {
    PagedUnit x;
    x.seq = u / p.row_tiles;
    x.row0 = (u - x.seq * p.row_tiles) * R;
    if constexpr (MODE == kShared) {  // of a group: its tokens lie one after the other, its pages are the first sequence's
        const int first = __ldg(p.group_start + x.seq), last = __ldg(p.group_start + x.seq + 1);
        const bool good = first >= 0 && last >= first && last <= p.kv.nseq;
        const int a = good ? __ldg(p.start + first) : 0, b = good ? __ldg(p.start + last) : 0;
        const int n = a < 0 || b > p.tokens || b < a ? 0 : b - a;
        x.len = prefix_rows(p, x.seq);
        x.seq = min(max(first, 0), p.kv.nseq - 1);
        x.tok0 = a;
        x.fresh = 0;
        x.rows = min(max(min(n, p.max_new) * p.group - x.row0, 0), R);
        x.end = x.rows == 0 ? 0 : x.len;
        if (x.end == 0) x.rows = 0;
        x.from = 0;
        return x;
    }
    x.len = p.kv.length(x.seq);
    x.from = 0;
    if constexpr (MODE == kOwn) {
        x.from = prefix_rows(p, paged_group_of(p, x.seq));
        x.len = max(x.len, x.from);
    }
    const int a = __ldg(p.start + x.seq), b = __ldg(p.start + x.seq + 1);
    x.tok0 = a;
    const int n = a < 0 || b > p.tokens || b < a ? 0 : b - a;  // (tokens that the arrays do not have)
    x.fresh = min(n, p.kv.rows - x.len);
    x.rows = min(max(min(n, p.max_new) * p.group - x.row0, 0), R);
    const int last = (x.row0 + x.rows - 1) / p.group;  // its last token
    x.end = x.rows == 0 ? 0 : x.len + (p.mask ? x.fresh : min(x.fresh, last + 1));
    return x;
}

template <int R, int MODE>
__device__ __forceinline__ PagedUnit paged_unit(const PagedAttn &p, int u) { return paged_unit_of<MODE>(p, u, R); }

// Whether the t-th new token of a sequence sees position `pos`, pos < end of its unit.
__device__ __forceinline__ bool paged_sees(const PagedAttn &p, const PagedUnit &u, int t, int pos) {
    const int d = pos - u.len;
    if (d < 0) return true;
    if (d >= u.fresh) return false;
    if (!p.mask) return d <= t;
    return d < 64 * p.mask_words && ((__ldg(p.mask + (long long)(u.tok0 + t) * p.mask_words + (d >> 6)) >> (d & 63)) & 1);
}

// Inclusive sums of v over the block's threads in sums[], the total returned. sums: room for the threads and kShareMore more.
constexpr int kShareMore = 34;  // one per warp, and what find_share() found
template <int THREADS>
__device__ __forceinline__ long long block_scan(int v, long long *sums) {
    long long *of_warp = sums + THREADS;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    long long s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == 31) of_warp[w] = s;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; i++) {
        if (i < w) before += of_warp[i];
        total += of_warp[i];
    }
    sums[threadIdx.x] = s + before;
    __syncthreads();
    return total;
}

template <int TILE, int MODE>
__device__ __forceinline__ int unit_tiles(const PagedUnit &u) { return MODE == kOwn ? (max(u.end - u.from, 0) + TILE - 1) / TILE : (u.end + TILE - 1) / TILE; }

// Says where the parts of an item lie that CTA `cta` has tiles t0 .. t1 - 1 of, its `slot`-th (0, 1) part if it does not have all of them.
template <int MODE>
__device__ __forceinline__ void note_span(const PagedAttn &p, int unit, int head, int t0, int t1, int tiles, int cta, int slot) {
    const long long item = (long long)unit * p.kv.nkv + head;
    int *span = p.spans + 2 * item;
    if (t0 == 0) span[0] = t1 < tiles ? 2 * cta + slot : whole_items<MODE>() ? -1 : (int)(p.whole_slot + item);
    if (t1 == tiles) span[1] = cta;
}

// The slot of a CTA's part of an item, its `slot`-th if it does not have all of it.
template <int MODE>
__device__ __forceinline__ size_t part_slot(const PagedAttn &p, int unit, int head, int t0, int t1, int tiles, int cta, int slot) {
    if (!whole_items<MODE>() && t0 == 0 && t1 == tiles) return p.whole_slot + (size_t)unit * p.kv.nkv + head;
    return (size_t)cta * 2 + slot;
}

// A row's weight of a position is 2^(score + norm): minus its maximum and the logarithm of its sum of weights, -inf where it sees nothing.
__device__ __forceinline__ float row_norm(float2 ml) { return ml.y > 0.0f ? -(ml.x + log2f(ml.y)) : ml.y == 0.0f ? -INFINITY : ml.y; }
// Adds to the sum of a position of a unit's sequence; a new row's sum starts with this call.
__device__ __forceinline__ void add_sum(const PagedAttn &p, const PagedUnit &u, int head, int pos, float v, bool first = true) {
    if (pos >= p.sum_cols) return;
    float *at = p.sums + u.seq * p.sum_seq + head * p.sum_head + pos;
    *at = first && pos >= u.len ? v : *at + v;
}

// Where a CTA's share starts.
struct Share {
    long long from, to;  // places in the list of all tiles
    int unit, head, tile;
};

// No share is empty: CTAs without a tile of their own have none, and leave no parts.
__device__ __forceinline__ int share_count(long long total, int ctas) { return (int)min((long long)ctas, total); }
// floor(total * c / n); n at most 2^15
__device__ __forceinline__ long long share_at(long long total, int n, int c) {
    if (c >= n) return total;
    const long long q = total >> 32 ? total / n : (long long)((uint32_t)total / (uint32_t)n);
    return q * c + (uint32_t)((int)(total - q * n) * c) / (uint32_t)n;
}

// LONG: of the units with more than `above` tiles alone, for CTA `cta` of `ctas`.
template <int R, int TILE, int THREADS, int MODE, bool LONG = false>
__device__ __forceinline__ Share find_share(const PagedAttn &p, int units, int ctas, long long *sums, PagedUnit &at, int above = 0, int cta = blockIdx.x) {
    int *found = reinterpret_cast<int *>(sums + THREADS + 32);  // unit, head, tile
    Share s;
    long long total = 0, before = 0;
    s.from = s.to = 0;
    s.unit = s.head = s.tile = 0;
    const bool once = units <= THREADS;  // the first pass over the units has all that the second one needs
    int n = 0;
#pragma unroll 1
    for (int pass = 0; pass < 2; pass++) {
#pragma unroll 1
        for (int u0 = 0; u0 < units; u0 += THREADS) {
            const int u = u0 + threadIdx.x;
            long long all = total;
            if (pass == 0 || !once) {
                n = u < units ? unit_tiles<TILE, MODE>(paged_unit<R, MODE>(p, u)) : 0;
                if (LONG && n <= above) n = 0;
                all = block_scan<THREADS>(n, sums);
            }
            if (pass == 0) {
                total += all;
                continue;
            }
            const long long a = (before + sums[threadIdx.x] - n) * p.kv.nkv;
            if (n > 0 && s.from >= a && s.from < a + (long long)n * p.kv.nkv) {
                const int d = (int)(s.from - a);
                found[0] = u;
                found[1] = d / n;
                found[2] = d % n;
            }
            before += all;
            if (before * p.kv.nkv > s.from) break;
        }
        if (pass == 0) {
            const long long tiles = total * p.kv.nkv;
            const int shares = share_count(tiles, ctas);
            s.from = share_at(tiles, shares, cta);
            s.to = share_at(tiles, shares, cta + 1);
            if (s.from >= s.to) return s;
        }
    }
    __syncthreads();
    s.unit = found[0];
    s.head = found[1];
    s.tile = found[2];
    at = paged_unit<R, MODE>(p, s.unit);
    __syncthreads();  // everyone has read found[]: `sums` may lie where the caller's warps, not all at a time, write next
    return s;
}

// The same by every warp for itself, for up to 32 units: a lane per unit, no synchronisation of the block.
template <int R, int TILE, int MODE>
__device__ __forceinline__ Share warp_share(const PagedAttn &p, int units, int ctas, PagedUnit &at) {
    const int lane = threadIdx.x & 31;
    PagedUnit u = paged_unit<R, MODE>(p, min(lane, units - 1));
    const int n = lane < units ? unit_tiles<TILE, MODE>(u) : 0;  // (32 sequences of 2^31 rows in tiles of 64: 2^30)
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += t;
    }
    const int all = __shfl_sync(0xffffffffu, sum, 31);
    Share s;
    const long long total = (long long)all * p.kv.nkv;
    const int shares = share_count(total, ctas);
    s.from = share_at(total, shares, blockIdx.x);
    s.to = share_at(total, shares, blockIdx.x + 1);
    s.unit = s.head = s.tile = 0;
    const long long a = (long long)(sum - n) * p.kv.nkv;
    const unsigned mine = __ballot_sync(0xffffffffu, n > 0 && s.from >= a && s.from < a + (long long)n * p.kv.nkv);
    if (s.from < s.to) {
        s.unit = __ffs(mine) - 1;
        const int d = (int)(s.from - a);
        s.head = __shfl_sync(0xffffffffu, n > 0 ? d / n : 0, s.unit);
        s.tile = __shfl_sync(0xffffffffu, n > 0 ? d % n : 0, s.unit);
    }
    at.seq = __shfl_sync(0xffffffffu, u.seq, s.unit);
    at.row0 = __shfl_sync(0xffffffffu, u.row0, s.unit);
    at.rows = __shfl_sync(0xffffffffu, u.rows, s.unit);
    at.tok0 = __shfl_sync(0xffffffffu, u.tok0, s.unit);
    at.len = __shfl_sync(0xffffffffu, u.len, s.unit);
    at.fresh = __shfl_sync(0xffffffffu, u.fresh, s.unit);
    at.end = __shfl_sync(0xffffffffu, u.end, s.unit);
    at.from = MODE == kOwn ? __shfl_sync(0xffffffffu, u.from, s.unit) : 0;
    return s;
}

// CTAs of a tcgen05 launch for the shared rows beside which the own rows are read by others: as many as make both end together, by what there is of both in this call (what a
// host knows, the longest sequence and the longest prefix, says little of either where they are not all alike). In SM microseconds: a tile of 128 positions 4 (256 rows) or 2.1
// (128) and 2 for a CTA's start; 55 own rows of a KV head one, whatever the heads' width. Fitted to 36 calls (16 to 64 sequences behind 2048 to 16000 rows, heads of 64 and 128, own rows alike and
// spread) with 12 .. 148 CTAs each: 4 % above the best number of CTAs on average, 17 % at most. (64 sequences of 700 rows of their own behind 8192: 112 us with 12 CTAs, 60 with 36, 62 with 74, 80 with 148.)
template <int R, int TILE, int THREADS>
__device__ __forceinline__ int shared_ctas_beside(const PagedAttn &p, long long *sums) {
    float tiles = 0.0f, rows = 0.0f;
    // (Every sequence counts, with new tokens or without, and every group as one of max_group_new tokens: one latency of loads. Which group a sequence is in and how many
    // tokens a group has would be chains of them, 2 us.)
    for (int i = threadIdx.x; i < max(p.kv.nseq, p.groups); i += THREADS) {
        const int len = i < p.kv.nseq ? p.kv.length(i) : 0, g = min(i, p.groups - 1);
        const int n = max(__ldg(p.group_start + g + 1) - __ldg(p.group_start + g), 0), prefix = prefix_rows(p, g);
        rows += len;
        if (i >= p.groups || n == 0) continue;
        rows -= (float)n * prefix;
        tiles += (float)p.row_tiles * ((prefix + TILE - 1) / TILE);
    }
    float2 *of_warp = reinterpret_cast<float2 *>(sums);
    const float2 mine = make_float2(warp_sum(tiles), warp_sum(rows));
    if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = mine;
    __syncthreads();
    tiles = rows = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) tiles += of_warp[w].x, rows += of_warp[w].y;
    __syncthreads();  // (`sums` is written again)
    const float shared = tiles * p.kv.nkv * (R == 256 ? 4.0f : 2.1f), own = max(rows, 0.0f) * p.kv.nkv * (1 / 55.0f);
    int lo = 1, hi = p.ctas;  // fewer CTAs leave more time and more SMs for the own rows
    while (lo < hi) {
        const int c = (lo + hi) / 2;
        if ((p.ctas - c) * (2.0f + shared / c) > own) lo = c + 1;
        else hi = c;
    }
    return lo;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool there) {  // zeros where there is no source
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A row whose sums are not finite, from the positions it sees alone: on the tensor cores a weight of zero times an infinite or missing value of a
// position that the row does not see is a NaN. A warp, 32 positions at a time, one a lane for the scores; o: this lane's columns (lane, lane + 32, ...).
template <bool BF16, int HD>
__device__ __noinline__ void plain_row(const PagedAttn &p, const PagedUnit &u, int head, int r, int from, int to, float *o, float &m, float &l) {
    const int lane = threadIdx.x & 31, t = (u.row0 + r) / p.group, h = head * p.group + (u.row0 + r) % p.group;
    const uint16_t *q = p.q + (u.tok0 + t) * p.qs + (long long)h * HD;
    const uint16_t *kc = p.kc + (long long)head * p.kv.page * HD, *vc = p.vc + (long long)head * p.kv.page * HD + lane;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 32; i++) o[i] = 0.0f;
#pragma unroll 1
    for (int left = to - from; left > 0; left -= 32) {
        const int pos = to - left + lane;
        const long long at = lane < left && paged_sees(p, u, t, pos) ? p.kv.row_of(u.seq, pos) : -1;
        float s = -INFINITY;
        if (at >= 0) {
            float d = 0.0f;
#pragma unroll 4
            for (int c = 0; c < HD; c += 8) {
                const uint4 a = *reinterpret_cast<const uint4 *>(q + c), b = *reinterpret_cast<const uint4 *>(kc + at + c);
                const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = unpack16<BF16>(x[j]), g = unpack16<BF16>(y[j]);
                    d = fmaf(f.x, g.x, d);
                    d = fmaf(f.y, g.y, d);
                }
            }
            s = d * p.scale2;
        }
        const unsigned seen = __ballot_sync(0xffffffffu, !(s == -INFINITY));
        if (seen == 0) continue;
        const float m_new = fmaxf(m, warp_max(s)), corr = m == m_new ? 1.0f : ex2(m - m_new), w = s == -INFINITY ? 0.0f : ex2(s - m_new);
        m = m_new;
        l = l * corr + warp_sum(w);
#pragma unroll
        for (int i = 0; i < HD / 32; i++) o[i] *= corr;
#pragma unroll 1
        for (int j0 = 0; j0 < 32; j0 += 4) {
            if (!(seen >> j0 & 15u)) continue;
            float x[4][HD / 32];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const long long from_row = __shfl_sync(0xffffffffu, at, j0 + j);
#pragma unroll
                for (int i = 0; i < HD / 32; i++) x[j][i] = seen >> (j0 + j) & 1u ? one16<BF16>(vc + from_row + 32 * i) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float f = __shfl_sync(0xffffffffu, w, j0 + j);
#pragma unroll
                for (int i = 0; i < HD / 32; i++) o[i] = fmaf(f, x[j][i], o[i]);
            }
        }
    }
}

// The sum of a position's weights over the rows of a unit, from queries and keys: a position a lane (-1: none), rows' norms in `norms`. For positions that a
// call has no room for the scores of.
template <bool BF16, int HD>
__device__ __noinline__ float plain_sum(const PagedAttn &p, const PagedUnit &u, int head, int pos, const float *norms) {
    const long long at = pos >= 0 && pos < u.end ? p.kv.row_of(u.seq, pos) : -1;
    const uint16_t *kc = p.kc + (long long)head * p.kv.page * HD + (at < 0 ? 0 : at);
    float v = 0.0f;
#pragma unroll 1
    for (int r = 0; r < u.rows; r++) {
        const int t = (u.row0 + r) / p.group, h = head * p.group + (u.row0 + r) % p.group;
        if (at < 0 || !paged_sees(p, u, t, pos)) continue;
        const uint16_t *q = p.q + (u.tok0 + t) * p.qs + (long long)h * HD;
        float d = 0.0f;
#pragma unroll 4
        for (int c = 0; c < HD; c += 8) {
            const uint4 a = *reinterpret_cast<const uint4 *>(q + c), b = *reinterpret_cast<const uint4 *>(kc + c);
            const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = unpack16<BF16>(x[j]), g = unpack16<BF16>(y[j]);
                d = fmaf(f.x, g.x, d);
                d = fmaf(f.y, g.y, d);
            }
        }
        v += ex2(fmaf(d, p.scale2, norms[r]));
    }
    return v;
}

// The sum `v` of a position's weights from kept scores, where it is not a number: a row with such a sum of weights is one wherever its scores are, at positions too that it does
// not see. Those that all rows see stay, new rows and what is not there are taken from the rows that see them alone.
template <bool BF16, int HD>
__device__ __forceinline__ float seen_sum(const PagedAttn &p, const PagedUnit &u, int head, int pos, const float *norms, float v) {
    return v == v || (pos < u.len && p.kv.row_of(u.seq, pos) >= 0) ? v : plain_sum<BF16, HD>(p, u, head, pos, norms);
}

// Row r of an item that a cut divides, by a warp, HD / 32 columns a lane. The parts of an item lie with the CTAs that its tiles fall to; a lane per part
// brings maxima and sums. (A block per row with the shares' divisions in loops took 25 us for 64 items of 104 rows.)
template <bool BF16, int R, int HD>
__device__ __forceinline__ void join_row(const PagedAttn &p, int item, int r) {
    constexpr int V = HD / 32;
    const int unit = item / p.kv.nkv, head = item - unit * p.kv.nkv, lane = threadIdx.x & 31;
    const int2 span = *reinterpret_cast<const int2 *>(p.spans + 2 * (long long)item);
    const PagedUnit u = paged_unit<R, kAttend>(p, unit);
    if (r >= u.rows || span.x < 0) return;  // (a unit without tiles has no rows)
    const size_t slot0 = span.x;
    const int c = span.x >> 1, parts = span.y - c + 1;
    auto at = [&](int i) { return (i == 0 ? slot0 : (size_t)(c + i) * 2) * R + r; };
    float M = -INFINITY, L = 0.0f, o[V];
#pragma unroll
    for (int j = 0; j < V; j++) o[j] = 0.0f;
    for (int i0 = 0; i0 < parts; i0 += 32) {
        const float2 x = i0 + lane < parts ? p.part_ml[at(i0 + lane)] : make_float2(-INFINITY, 0.0f);
        const float top = fmaxf(M, warp_max(x.x)), corr = M == top ? 1.0f : ex2(M - top);
        const float f = x.x == -INFINITY && x.y == 0.0f ? 0.0f : ex2(x.x - top);  // (nothing seen in this part)
        M = top;
        L = L * corr + warp_sum(x.y * f);
#pragma unroll
        for (int j = 0; j < V; j++) o[j] *= corr;
        const int m = min(32, parts - i0);
#pragma unroll 4
        for (int i = 0; i < m; i++) {
            const float *src = p.part_o + at(i0 + i) * HD + lane * V;
            const float g = __shfl_sync(0xffffffffu, f, i);
            float v[V];
            if constexpr (V == 2) *reinterpret_cast<float2 *>(v) = *reinterpret_cast<const float2 *>(src);
            else
#pragma unroll
                for (int j = 0; j < V; j += 4) *reinterpret_cast<float4 *>(v + j) = *reinterpret_cast<const float4 *>(src + j);
#pragma unroll
            for (int j = 0; j < V; j++) o[j] += g == 0.0f ? 0.0f : v[j] * g;
        }
    }
    const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
    const int t = (u.row0 + r) / p.group, g = (u.row0 + r) % p.group;
    uint32_t *dst = reinterpret_cast<uint32_t *>(p.out + (u.tok0 + t) * p.os + (long long)(head * p.group + g) * HD + lane * V);
#pragma unroll
    for (int j = 0; j < V; j += 2) dst[j / 2] = pack16<BF16>(o[j] * inv, o[j + 1] * inv);
}
// Many rows of a KV head on the tcgen05 tensor cores (paged_attn_tc.cu): rows of a tile for so many rows of a sequence, 0 where the
// kernel of paged_attn.cu is the one to use; CTAs = SMs.
int paged_tc_rows(int hd, long long rows);
int paged_tc_launch(const Device *dev, const PagedAttn &p, bool bf16, int rows, int units, cudaStream_t st);

// Rows that no sequence passes.
int attn_length(const PagedView &v, int max_len);
// What calls have in common: heads and new tokens checked; all arguments checked and p filled in but for the plan (empty: there is nothing to do).
int attn_check(const im_paged_kv *kv, int num_heads, int max_new);
int attn_args(im_device *dev, const im_paged_kv *kv, int layer, const void *q_dev, int64_t q_stride, void *out_dev, int64_t out_stride, int num_heads,
              const int *token_start_dev, int num_tokens, int max_new, const uint64_t *mask_dev, int mask_words, float scale, int max_len, PagedAttn *p, bool *empty);

// The kernel of paged_attn_tc.cu with the sums of a part as its result (paged_prefix.cu): MODE kShared or kOwn; no join.
int paged_tc_part_launch(const Device *dev, const PagedAttn &p, bool bf16, int mode, int rows, int units, cudaStream_t st);
// Adds the parts i, i + step, ... of a row, maxima and sums of weights, at `ml`: slots of R rows. Eight are requested together.
__device__ __forceinline__ float2 row_parts(const float2 *ml, int2 span, int R, int r, int i, int step) {
    const int c = span.x >> 1, parts = span.y - c + 1;
    float M = -INFINITY, L = 0.0f;
#pragma unroll 1
    for (; i < parts; i += 8 * step) {
        float2 x[8];
        float top = M;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int at = min(i + k * step, parts - 1);
            x[k] = ml[(at == 0 ? (size_t)span.x : (size_t)(c + at) * 2) * R + r];
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (i + k * step >= parts) x[k] = make_float2(-INFINITY, 0.0f);
            top = fmaxf(top, x[k].x);
        }
        L = M == top ? L : L * ex2(M - top);
#pragma unroll
        for (int k = 0; k < 8; k++) L += x[k].x == -INFINITY && x[k].y == 0.0f ? 0.0f : x[k].y * ex2(x[k].x - top);
        M = top;
    }
    return make_float2(M, L);
}
// Attention and the norms of every row's weights (paged_weights.cu): where `cluster` is not zero, the sums too. joins: with the join of what the cuts divide (tcgen05: always).
int paged_weigh_launch(const Device *dev, const PagedAttn &p, bool bf16, int units, int cluster, bool joins, cudaStream_t st);
int paged_tc_weigh_launch(const Device *dev, const PagedAttn &p, bool bf16, int rows, int units, cudaStream_t st);
struct AttnPlan {
    int rows, tile, row_tiles, units, ctas;
    int cluster;  // CTAs per item that join in the launch; 0: shares
    size_t bytes;
};
AttnPlan attn_plan(const Device *dev, int nseq, int nkv, int hd, int group, int max_new, int max_len);
// A plan in the arguments of a launch, its scratch from `at` on.
void attn_lay_out(PagedAttn *p, const AttnPlan &plan, int max_len, void *at);
// Sums of weighted values that a share of paged_attn_tc.cu leaves: four columns of all rows after another, since a warp that writes (and one that joins) has a row per lane.
template <int R>
__device__ __forceinline__ float *tc_part(float *part_o, size_t slot, int hd, int row, int col) { return part_o + (slot * (hd / 4) + col / 4) * (R * 4) + row * 4 + col % 4; }

}  // namespace im
