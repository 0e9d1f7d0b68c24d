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
};

// A unit: a tile of rows (token, query head of the KV head) of one sequence, rows token-major.
struct PagedUnit {
    int seq, row0, rows;      // first row among the sequence's; rows of it that exist
    int tok0;                 // the sequence's first new token
    int len, fresh;           // rows before the new ones; new ones that lie in the table
    int end;                  // no row of the unit sees a position from here on
};

template <int R>
__device__ __forceinline__ PagedUnit paged_unit(const PagedAttn &p, int u) {
    PagedUnit x;
    x.seq = u / p.row_tiles;
    x.row0 = (u - x.seq * p.row_tiles) * R;
    x.len = p.kv.length(x.seq);
    const int a = __ldg(p.start + x.seq), b = __ldg(p.start + x.seq + 1);
    x.tok0 = a;
    const int n = a < 0 || b > p.tokens || b < a ? 0 : b - a;  // (tokens that the arrays do not have)
    x.fresh = min(n, p.kv.rows - x.len);
    x.rows = min(max(min(n, p.max_new) * p.group - x.row0, 0), R);
    const int last = (x.row0 + x.rows - 1) / p.group;  // its last token
    x.end = x.rows == 0 ? 0 : x.len + (p.mask ? x.fresh : min(x.fresh, last + 1));
    return x;
}

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

template <int TILE>
__device__ __forceinline__ int unit_tiles(const PagedUnit &u) { return (u.end + TILE - 1) / TILE; }

// Says where the parts of an item lie that CTA `cta` has tiles t0 .. t1 - 1 of, its `slot`-th (0, 1) part if it does not have all of them.
__device__ __forceinline__ void note_span(const PagedAttn &p, int unit, int head, int t0, int t1, int tiles, int cta, int slot) {
    int *span = p.spans + 2 * ((long long)unit * p.kv.nkv + head);
    if (t0 == 0) span[0] = t1 == tiles ? -1 : 2 * cta + slot;
    if (t1 == tiles) span[1] = cta;
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

template <int R, int TILE, int THREADS>
__device__ __forceinline__ Share find_share(const PagedAttn &p, int units, long long *sums, PagedUnit &at) {
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
                n = u < units ? unit_tiles<TILE>(paged_unit<R>(p, u)) : 0;
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
            const int shares = share_count(tiles, p.ctas);
            s.from = share_at(tiles, shares, blockIdx.x);
            s.to = share_at(tiles, shares, blockIdx.x + 1);
            if (s.from >= s.to) return s;
        }
    }
    __syncthreads();
    s.unit = found[0];
    s.head = found[1];
    s.tile = found[2];
    at = paged_unit<R>(p, s.unit);
    __syncthreads();  // everyone has read found[]: `sums` may lie where the caller's warps, not all at a time, write next
    return s;
}

// The same by every warp for itself, for up to 32 units: a lane per unit, no synchronisation of the block.
template <int R, int TILE>
__device__ __forceinline__ Share warp_share(const PagedAttn &p, int units, PagedUnit &at) {
    const int lane = threadIdx.x & 31;
    PagedUnit u = paged_unit<R>(p, min(lane, units - 1));
    const int n = lane < units ? unit_tiles<TILE>(u) : 0;  // (32 sequences of 2^31 rows in tiles of 64: 2^30)
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += t;
    }
    const int all = __shfl_sync(0xffffffffu, sum, 31);
    Share s;
    const long long total = (long long)all * p.kv.nkv;
    const int shares = share_count(total, p.ctas);
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
    return s;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool there) {  // zeros where there is no source
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
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

// Many rows of a KV head on the tcgen05 tensor cores (paged_attn_tc.cu): rows of a tile for so many rows of a sequence, 0 where the
// kernel of paged_attn.cu is the one to use; CTAs = SMs.
int paged_tc_rows(int hd, long long rows);
int paged_tc_launch(const Device *dev, const PagedAttn &p, bool bf16, int rows, int units, cudaStream_t st);

}  // namespace im
