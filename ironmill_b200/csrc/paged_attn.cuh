// Attention over a paged cache: what its kernels share (paged_attn.cu).
#pragma once
#include "paged.cuh"

namespace im {

struct PagedAttn {
    PagedView kv;
    const uint16_t *kc, *vc;  // of the layer
    const uint16_t *q;
    uint16_t *out;
    long long qs, os;
    const int *start;
    const uint64_t *mask;
    int mask_words, nh, group, tokens, max_new;
    float scale2;             // scale / ln 2: scores in powers of two
    int row_tiles;            // row tiles of a sequence: ceil(max_new * group / rows of a tile)
    int ctas;                 // CTAs of the attention kernel
    float *part_o;            // [ctas, 2, rows of a tile, head_dim]: sums of weighted values
    float2 *part_ml;          // [ctas, 2, rows of a tile]: maximum, sum of weights
    long long *first;         // [units + 1]: tiles of one KV head before a unit
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

}  // namespace im
