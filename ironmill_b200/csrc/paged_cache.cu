// A paged cache of keys and values: appending with rotation (and norms), keeping the accepted path of a drafted tree, reordering the beams of a search.
// All of them move rows and compute next to nothing: HBM bounds them where they are large, the chain of lookups (sequence of a
// token -> its length -> its page) where they are small. 16 bytes a lane and access (8 where keys and queries are normed, 2 where they are and rotary_dim is no multiple of 8).
#include <limits.h>

#include <algorithm>

#include "paged.cuh"

namespace im {

int paged_view(const im_paged_kv *kv, int layer, PagedView *out) {
    IM_REQUIRE(kv, "kv is NULL");
    IM_REQUIRE(kv->dtype == IM_DTYPE_F16 || kv->dtype == IM_DTYPE_BF16, "paged caches hold fp16 or bf16 (got dtype %d)", kv->dtype);
    IM_REQUIRE(kv->num_layers > 0 && kv->num_pages > 0 && kv->num_kv_heads > 0 && kv->page_size > 0 && kv->num_seqs >= 0 && kv->table_width > 0, "bad shape of a paged cache");
    IM_REQUIRE(kv->head_dim > 0 && kv->head_dim % 8 == 0 && kv->head_dim <= 256, "head_dim has to be a multiple of 8 up to 256 (got %d)", kv->head_dim);
    IM_REQUIRE(kv->k_dev && kv->v_dev && (kv->num_seqs == 0 || (kv->page_table_dev && kv->seq_len_dev)), "a pointer of the paged cache is NULL");
    IM_REQUIRE(kv->k_dev != kv->v_dev, "keys and values lie in the same place");
    IM_REQUIRE(aligned16(kv->k_dev) && aligned16(kv->v_dev), "keys and values have to be 16-byte aligned");
    IM_REQUIRE((long long)kv->table_width * kv->page_size <= INT_MAX, "a sequence of %lld rows is too long", (long long)kv->table_width * kv->page_size);
    const long long most = 1ll << 46;
    IM_REQUIRE((long long)kv->num_kv_heads * kv->page_size <= most / 256 / kv->num_pages / kv->num_layers, "bad shape of a paged cache");
    const long long block = (long long)kv->num_kv_heads * kv->page_size * kv->head_dim;
    PagedView v;
    v.page_stride = kv->page_stride ? kv->page_stride : block;
    v.layer_stride = kv->layer_stride ? kv->layer_stride : v.page_stride * kv->num_pages;
    IM_REQUIRE(v.page_stride % 8 == 0 && v.layer_stride % 8 == 0 && v.page_stride >= block && v.page_stride <= most / kv->num_pages && v.layer_stride > 0 &&
                   v.layer_stride <= most / kv->num_layers,
               "strides of pages and layers have to be multiples of 8 elements that hold them");
    IM_REQUIRE(kv->num_layers == 1 || v.layer_stride >= (kv->num_pages - 1) * v.page_stride + block ||
                   (v.layer_stride >= block && (kv->num_pages == 1 || v.page_stride >= (kv->num_layers - 1) * v.layer_stride + block)),
               "pages of different layers overlap");
    v.table_stride = kv->table_stride ? kv->table_stride : kv->table_width;
    IM_REQUIRE(v.table_stride >= kv->table_width, "rows of the page table overlap");
    IM_REQUIRE(layer < kv->num_layers, "layer %d of %d", layer, kv->num_layers);
    v.layers = kv->num_layers;
    v.pages = kv->num_pages;
    v.nkv = kv->num_kv_heads;
    v.page = kv->page_size;
    v.hd = kv->head_dim;
    v.nseq = kv->num_seqs;
    v.width = kv->table_width;
    v.rows = kv->table_width * kv->page_size;
    v.table = kv->page_table_dev;
    v.len = kv->seq_len_dev;
    *out = v;
    return IM_OK;
}

int paged_device(const im_device *dev) {
    IM_REQUIRE(dev, "dev is NULL");
    int current = -1;
    IM_CUDA_CHECK(cudaGetDevice(&current));
    IM_REQUIRE(current == dev->ordinal, "the handle's device %d is not the current one (%d)", dev->ordinal, current);
    return IM_OK;
}

namespace {

// ------------------------------------------------------------------------------------------------ append
struct Append {
    PagedView kv;
    uint16_t *kc, *vc;  // of the layer
    const uint16_t *k, *v, *q;
    uint16_t *qo;
    long long ks, vs, qs, qos;
    const int *start, *pos;
    const void *cosc, *sinc;
    int nh, max_pos, rot;
};

// Four entries of a table at a multiple of four: rows have head_dim / 2 of them, a multiple of four.
template <bool F32>
__device__ __forceinline__ void angles4(const void *table, long long at, float *out) {
    if (F32) {
        *reinterpret_cast<float4 *>(out) = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(table) + at));
    } else {
        const uint2 u = __ldg(reinterpret_cast<const uint2 *>(static_cast<const __half *>(table) + at));
        const float2 lo = unpack16<false>(u.x), hi = unpack16<false>(u.y);
        out[0] = lo.x; out[1] = lo.y; out[2] = hi.x; out[3] = hi.y;
    }
}

// A block per token; `lanes` lanes (the power of two from head_dim / 8 up) hold a head, eight columns each, and walk the heads with the same
// cosines and sines. The first heads of a thread are requested before the lookups of the token's place (its sequence, the sequence's length,
// its page): one latency for the loads, one chain for the place, hidden by the other blocks of the SM.
// FORM: 0 nothing is rotated; 1 halves, a column's partner a whole number of lanes away; 2 neighbours; 3 halves, partners anywhere.
// Blocks of 64 threads where there are many (8 x 1900 tokens of 48 heads: 59 us in blocks of 256, 51 of 128, 49 of 64), of 256 where a block more or less
// costs nothing (32 tokens: 3.3 us, 6.4 in blocks of 64).
constexpr int kAppendThreads = 256, kAppendSmall = 64;
constexpr int kAppendMost = 1 << 20;  // heads of a call
constexpr int kAppendHeads = 3;  // heads that a thread holds at a time

template <bool BF16, int FORM, bool F32>
__global__ void __launch_bounds__(kAppendThreads, FORM == 3 ? 2 : 5) paged_append_kernel(const __grid_constant__ Append a, int lanes) {
    pdl_trigger();
    pdl_wait();
    const int token = blockIdx.x, tid = threadIdx.x;
    const int c = tid & (lanes - 1), first = tid / lanes, per = blockDim.x / lanes;
    const int hd = a.kv.hd, heads = a.nh + 2 * a.kv.nkv, d0 = 8 * c, half = a.rot / 2;
    const bool mine = d0 < hd;
    bool placed = false;
    long long at = -1;
    float cs[8], sn[8];
#pragma unroll 1
    for (int h0 = first; h0 - first < heads; h0 += per * kAppendHeads) {  // the same count for every lane of a warp
        uint4 x[kAppendHeads];
#pragma unroll
        for (int i = 0; i < kAppendHeads; i++) {
            const int h = h0 + i * per;
            x[i] = make_uint4(0, 0, 0, 0);
            if (mine && h < heads) {
                const uint16_t *src = h < a.nh ? a.q + token * a.qs + (long long)h * hd
                                               : h < a.nh + a.kv.nkv ? a.k + token * a.ks + (long long)(h - a.nh) * hd : a.v + token * a.vs + (long long)(h - a.nh - a.kv.nkv) * hd;
                x[i] = *reinterpret_cast<const uint4 *>(src + d0);
            }
        }
        if (!placed) {
            placed = true;
            const int lo = __ldg(a.start), hi = __ldg(a.start + a.kv.nseq);
            if (token < lo || token >= hi) return;
            const int seq = paged_seq_of(a.start, a.kv.nseq, token), place = token - __ldg(a.start + seq);
            const long long r = (long long)a.kv.length(seq) + place;
            if (place < 0 || r > INT_MAX) return;
            const int p = a.pos ? __ldg(a.pos + token) : (int)r;
            if (FORM > 0) {
                if ((unsigned)p >= (unsigned)a.max_pos) return;
                const long long row = (long long)p * (hd / 2);
                if (FORM == 1 && d0 < a.rot) {
                    const int e0 = d0 < half ? d0 : d0 - half;
                    angles4<F32>(a.cosc, row + e0, cs);
                    angles4<F32>(a.cosc, row + e0 + 4, cs + 4);
                    angles4<F32>(a.sinc, row + e0, sn);
                    angles4<F32>(a.sinc, row + e0 + 4, sn + 4);
                }
                if (FORM == 2 && mine) {
                    angles4<F32>(a.cosc, row + d0 / 2, cs);
                    angles4<F32>(a.sinc, row + d0 / 2, sn);
                }
                if (FORM == 3) {  // a chunk may hold the end of one half and the start of the other
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int d = d0 + i, e = d < half ? d : d - half;
                        cs[i] = sn[i] = 0.0f;
                        if (d < a.rot) {
                            cs[i] = F32 ? __ldg(static_cast<const float *>(a.cosc) + row + e) : __half2float(__ldg(static_cast<const __half *>(a.cosc) + row + e));
                            sn[i] = F32 ? __ldg(static_cast<const float *>(a.sinc) + row + e) : __half2float(__ldg(static_cast<const __half *>(a.sinc) + row + e));
                        }
                    }
                }
            }
            at = a.kv.row_of(seq, (int)r);
        }
#pragma unroll
        for (int i = 0; i < kAppendHeads; i++) {
            const int h = h0 + i * per;
            const bool is_v = h >= a.nh + a.kv.nkv;
            if (FORM > 0) {
                uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                float g[8];  // partners, where they are not in the same word
                if (FORM == 1) {
                    const int from = (threadIdx.x & 31 & ~(lanes - 1)) + ((c + (d0 < half ? half / 8 : lanes - half / 8)) & (lanes - 1));
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float2 t = unpack16<BF16>(__shfl_sync(0xffffffffu, w[j], from));
                        g[2 * j] = t.x;
                        g[2 * j + 1] = t.y;
                    }
                }
                if (FORM == 3) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int d = d0 + j, partner = d < half ? d + half : d - half;
                        g[j] = 0.0f;
                        if (mine && h < heads && !is_v && d < a.rot) {
                            const uint16_t *src = h < a.nh ? a.q + token * a.qs + (long long)h * hd : a.k + token * a.ks + (long long)(h - a.nh) * hd;
                            g[j] = one16<BF16>(src + partner);
                        }
                    }
                    __syncwarp();  // queries may be written over what was read
                }
                if (!is_v) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (d0 + 2 * j >= a.rot) continue;  // (rot is even: both columns of a word are rotated or neither is)
                        const float2 f = unpack16<BF16>(w[j]);
                        if (FORM == 2) {
                            w[j] = pack16<BF16>(f.x * cs[j] - f.y * sn[j], f.y * cs[j] + f.x * sn[j]);
                        } else {
                            const float y0 = d0 + 2 * j < half ? -g[2 * j] : g[2 * j], y1 = d0 + 2 * j + 1 < half ? -g[2 * j + 1] : g[2 * j + 1];
                            w[j] = pack16<BF16>(f.x * cs[2 * j] + y0 * sn[2 * j], f.y * cs[2 * j + 1] + y1 * sn[2 * j + 1]);
                        }
                    }
                }
                x[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (!mine || h >= heads) continue;
            if (h < a.nh) {
                *reinterpret_cast<uint4 *>(a.qo + token * a.qos + (long long)h * hd + d0) = x[i];
            } else if (at >= 0) {
                const int kvh = is_v ? h - a.nh - a.kv.nkv : h - a.nh;
                *reinterpret_cast<uint4 *>((is_v ? a.vc : a.kc) + at + (long long)kvh * a.kv.page * hd + d0) = x[i];
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ append with norms and several axes
//   y = x * rsqrt(mean(x^2) + eps) * w per head (keys and queries, each if it has weights), then pair i of y's columns turned by entry i of the table row
//   of position[axis of i]; f32 from the load to the one rounding at the end.
// The same blocks and lookups as above, but a lane owns both columns of its pairs (four of them: two words of 8 bytes, which lie side by side where
// neighbours belong together and half of rotary_dim apart where the halves do), so that rotation exchanges nothing between lanes, and every cosine and sine
// is loaded once instead of by both lanes of a pair. A token's weights, cosines and sines are multiplied once, a head
// is then two products and a factor an element, two elements at a time; its sum of squares is the only exchange, log2(lanes) shuffles.
// 8 prompts of up to 1900 tokens of 48 heads, three axes (260 MB): 57 us, 4.6 TB/s, 70 % of a copy; instructions issued in two of three clocks, and loads waited for, bound it (82 us with 16
// bytes a lane of both halves, partners by shuffles and a loop of shuffles). Blocks of 64 threads 57 us, of 32 as much, of 128 66, of 256 103; 32 tokens, in blocks of 256, 6 us.
constexpr int kAxes = 4;
struct AppendMore {
    const void *qn, *kn;  // weights or NULL
    int norm_f32, axes, neighbours;
    float eps, inv_dim;
    uint32_t axis[8];     // two bits a pair: 128 of them
};

// Where a token goes: the offset of its row in the cache (-1: it has none there) and the rows of the tables; false: it is left alone.
__device__ __forceinline__ bool append_place(const Append &a, const AppendMore &m, int token, long long &at, int (&pos)[kAxes]) {
    const int lo = __ldg(a.start), hi = __ldg(a.start + a.kv.nseq);
    if (token < lo || token >= hi) return false;
    const int seq = paged_seq_of(a.start, a.kv.nseq, token), place = token - __ldg(a.start + seq);
    const long long r = (long long)a.kv.length(seq) + place;
    if (place < 0 || r > INT_MAX) return false;
    bool there = true;
    if (a.rot > 0) {
#pragma unroll
        for (int k = 0; k < kAxes; k++) {
            pos[k] = k >= m.axes ? 0 : a.pos ? __ldg(a.pos + (long long)k * gridDim.x + token) : (int)r;
            there = there && (unsigned)pos[k] < (unsigned)a.max_pos;
        }
    }
    at = a.kv.row_of(seq, (int)r);
    return there;
}
// Cosines and sines of pairs e0 .. e0 + 3 (e0 a multiple of 4, below rotary_dim / 2), each from the row of its axis: all four from the first one's, and those of other axes again.
template <bool F32>
__device__ __forceinline__ void append_angles(const Append &a, const AppendMore &m, const int (&pos)[kAxes], int e0, float *cs, float *sn) {
    const uint32_t axes = m.axis[e0 / 16 & 7] >> (2 * (e0 & 15)) & 255u;  // (sixteen pairs a word)
    auto row = [&](uint32_t k) { return (long long)(k == 0 ? pos[0] : k == 1 ? pos[1] : k == 2 ? pos[2] : pos[3]) * (a.kv.hd / 2); };
    const long long at = row(axes & 3);
    angles4<F32>(a.cosc, at + e0, cs);
    angles4<F32>(a.sinc, at + e0, sn);
    if (axes == (axes & 3) * 0x55u) return;
#pragma unroll
    for (int j = 1; j < 4; j++) {
        const long long e = row(axes >> (2 * j) & 3) + e0 + j;
        cs[j] = F32 ? __ldg(static_cast<const float *>(a.cosc) + e) : __half2float(__ldg(static_cast<const __half *>(a.cosc) + e));
        sn[j] = F32 ? __ldg(static_cast<const float *>(a.sinc) + e) : __half2float(__ldg(static_cast<const __half *>(a.sinc) + e));
    }
}
template <bool BF16>
__device__ __forceinline__ float norm_weight(const void *w, int f32, int d) {
    return !w ? 1.0f : f32 ? __ldg(static_cast<const float *>(w) + d) : one16<BF16>(static_cast<const uint16_t *>(w) + d);
}
// Four norm weights from column d on, a multiple of 4.
template <bool BF16>
__device__ __forceinline__ void weights4(const void *w, int f32, int d, float *out) {
    if (!w) {
#pragma unroll
        for (int j = 0; j < 4; j++) out[j] = 1.0f;
    } else if (f32) {
        *reinterpret_cast<float4 *>(out) = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(w) + d));
    } else {
        const uint2 u = __ldg(reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(w) + d));
        const float2 lo = unpack16<BF16>(u.x), hi = unpack16<BF16>(u.y);
        out[0] = lo.x; out[1] = lo.y; out[2] = hi.x; out[3] = hi.y;
    }
}

// rotary_dim a multiple of 8: the four pairs of a lane are turned or none is.
constexpr int kNormedHeads = 4;
template <bool BF16, bool NB, bool F32, int LANES>
__global__ void __launch_bounds__(kAppendThreads, 4) paged_append_normed_kernel(const __grid_constant__ Append a, const __grid_constant__ AppendMore m) {
    pdl_trigger();
    pdl_wait();
    const int token = blockIdx.x, tid = threadIdx.x;
    const int c = tid % LANES, first = tid / LANES, per = blockDim.x / LANES;
    const int hd = a.kv.hd, half = a.rot / 2, e0 = 4 * c;
    const bool mine = 8 * c < hd, turned = e0 < half;
    const int colA = !NB && turned ? e0 : 2 * e0, colB = !NB && turned ? half + e0 : 2 * e0 + 4;
    uint2 x[kNormedHeads][2];
    auto load = [&](const uint16_t *src, int h0, int heads) {
#pragma unroll
        for (int i = 0; i < kNormedHeads; i++) {
            const int h = h0 + i * per;
            x[i][0] = x[i][1] = make_uint2(0, 0);
            if (mine && h < heads) {
                x[i][0] = *reinterpret_cast<const uint2 *>(src + h * hd + colA);
                x[i][1] = *reinterpret_cast<const uint2 *>(src + h * hd + colB);
            }
        }
    };
    const bool queries = a.nh > 0;
    const uint16_t *src = queries ? a.q + token * a.qs : a.k + token * a.ks;
    load(src, first, queries ? a.nh : a.kv.nkv);  // the first heads are requested before the lookups
    long long at;
    int pos[kAxes];
    if (!append_place(a, m, token, at, pos)) return;
    float cs[4], sn[4];
    if (turned && mine) append_angles<F32>(a, m, pos, e0, cs, sn);
    else
#pragma unroll
        for (int j = 0; j < 4; j++) cs[j] = 1.0f, sn[j] = 0.0f;
    // an element and its partner in the pair: y = (x C + partner S) r. Words A (0, 1) and B (2, 3) of two elements each; partners: the other word's, or (NB)
    // the word's own, exchanged
    auto turn = [&](const void *norm, const uint16_t *src, int heads, uint16_t *dst, long long dst_head, bool loaded) {
        uint64_t C[4], S[4];
        {
            float wa[4], wb[4];
            if (mine) {
                weights4<BF16>(norm, m.norm_f32, colA, wa);
                weights4<BF16>(norm, m.norm_f32, colB, wb);
            }
            if (NB) {
                C[0] = two(wa[0] * cs[0], wa[1] * cs[0]); C[1] = two(wa[2] * cs[1], wa[3] * cs[1]);
                C[2] = two(wb[0] * cs[2], wb[1] * cs[2]); C[3] = two(wb[2] * cs[3], wb[3] * cs[3]);
                S[0] = two(-wa[1] * sn[0], wa[0] * sn[0]); S[1] = two(-wa[3] * sn[1], wa[2] * sn[1]);
                S[2] = two(-wb[1] * sn[2], wb[0] * sn[2]); S[3] = two(-wb[3] * sn[3], wb[2] * sn[3]);
            } else {
                C[0] = two(wa[0] * cs[0], wa[1] * cs[1]); C[1] = two(wa[2] * cs[2], wa[3] * cs[3]);
                C[2] = two(wb[0] * cs[0], wb[1] * cs[1]); C[3] = two(wb[2] * cs[2], wb[3] * cs[3]);
                S[0] = two(-wb[0] * sn[0], -wb[1] * sn[1]); S[1] = two(-wb[2] * sn[2], -wb[3] * sn[3]);
                S[2] = two(wa[0] * sn[0], wa[1] * sn[1]); S[3] = two(wa[2] * sn[2], wa[3] * sn[3]);
            }
        }
#pragma unroll 1
        for (int h0 = first; h0 - first < heads; h0 += per * kNormedHeads) {  // the same count for every lane of a warp
            if (!loaded) load(src, h0, heads);
            loaded = false;
#pragma unroll
            for (int i = 0; i < kNormedHeads; i++) {
                const int h = h0 + i * per;
                if (h0 - first + i * per >= heads) break;  // (uniform)
                uint64_t X[4], P[4];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float2 lo = unpack16<BF16>(x[i][j].x), hi = unpack16<BF16>(x[i][j].y);
                    X[2 * j] = two(lo.x, lo.y);
                    X[2 * j + 1] = two(hi.x, hi.y);
                    if (NB) P[2 * j] = two(lo.y, lo.x), P[2 * j + 1] = two(hi.y, hi.x);
                }
                if (!NB) P[0] = X[2], P[1] = X[3], P[2] = X[0], P[3] = X[1];
                float r = 1.0f;
                if (norm) {
                    const float2 q = of_two(add_two(fma_two(X[0], X[0], mul_two(X[1], X[1])), fma_two(X[2], X[2], mul_two(X[3], X[3]))));
                    float sum = q.x + q.y;
                    #pragma unroll
                    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    r = rsqrtf(fmaf(sum, m.inv_dim, m.eps));
                }
                const uint64_t rr = two(r, r);
                uint32_t y[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint64_t v = mul_two(X[j], C[j]);
                    if (turned) v = fma_two(P[j], S[j], v);
                    const float2 f = of_two(mul_two(v, rr));
                    y[j] = pack16<BF16>(f.x, f.y);
                }
                if (mine && h < heads && dst) {
                    *reinterpret_cast<uint2 *>(dst + h * dst_head + colA) = make_uint2(y[0], y[1]);
                    *reinterpret_cast<uint2 *>(dst + h * dst_head + colB) = make_uint2(y[2], y[3]);
                }
            }
        }
    };
    const long long head = (long long)a.kv.page * hd;
    if (queries) turn(m.qn, src, a.nh, a.qo + token * a.qos, hd, true);
    turn(m.kn, a.k + token * a.ks, a.kv.nkv, at < 0 ? nullptr : a.kc + at, head, !queries);
    if (at < 0 || !mine) return;
    const uint16_t *v = a.v + token * a.vs + 8 * c;
    uint16_t *to = a.vc + at + 8 * c;
#pragma unroll 2
    for (int h = first; h < a.kv.nkv; h += per) *reinterpret_cast<uint4 *>(to + h * head) = *reinterpret_cast<const uint4 *>(v + h * hd);
}

// Any even rotary_dim, column by column: the columns behind the rotated ones are pairs of neighbours that are not turned. Loads and stores of 2 bytes bound it: the 8 prompts above with
// a rotary_dim of 100 137 us (2.4 times as long), 32 tokens 11.8 us a call as the others.
template <bool BF16, bool F32>
__global__ void __launch_bounds__(kAppendThreads) paged_append_odd_kernel(const __grid_constant__ Append a, const __grid_constant__ AppendMore m, int lanes) {
    pdl_trigger();
    pdl_wait();
    const int token = blockIdx.x, tid = threadIdx.x;
    const int c = tid & (lanes - 1), first = tid / lanes, per = blockDim.x / lanes;
    const int hd = a.kv.hd, heads = a.nh + 2 * a.kv.nkv, half = a.rot / 2, e0 = 4 * c;
    const bool mine = 8 * c < hd;
    auto column = [&](int i) {  // of pair e0 + i % 4, its first or (i >= 4) second one
        const int e = e0 + i % 4;
        return !m.neighbours && e < half ? e + (i / 4) * half : 2 * e + i / 4;
    };
    long long at;
    int pos[kAxes];
    if (!append_place(a, m, token, at, pos)) return;
    float cs[4], sn[4];
    if (e0 < half && mine) append_angles<F32>(a, m, pos, e0, cs, sn);
#pragma unroll 1
    for (int h = first; h - first < heads; h += per) {  // the same count for every lane of a warp
        const bool is_q = h < a.nh, is_v = h >= a.nh + a.kv.nkv, live = mine && h < heads;
        const uint16_t *src = is_q ? a.q + token * a.qs + (long long)h * hd : !is_v ? a.k + token * a.ks + (long long)(h - a.nh) * hd : a.v + token * a.vs + (long long)(h - a.nh - a.kv.nkv) * hd;
        uint16_t raw[8];
        float f[8], sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            raw[j] = live ? src[column(j)] : (uint16_t)0;
            f[j] = one16<BF16>(raw + j);
            sum = fmaf(f[j], f[j], sum);
        }
        for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (!live || (!is_q && at < 0)) continue;
        uint16_t *to = is_q ? a.qo + token * a.qos + (long long)h * hd : (is_v ? a.vc : a.kc) + at + (long long)(is_v ? h - a.nh - a.kv.nkv : h - a.nh) * a.kv.page * hd;
        const void *norm = is_q ? m.qn : m.kn;
        const float r = norm ? rsqrtf(fmaf(sum, m.inv_dim, m.eps)) : 1.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float p = f[j] * r * norm_weight<BF16>(norm, m.norm_f32, column(j)), q = f[j + 4] * r * norm_weight<BF16>(norm, m.norm_f32, column(j + 4));
            const bool turned = e0 + j < half;
            const float y = turned ? p * cs[j] - q * sn[j] : p, z = turned ? q * cs[j] + p * sn[j] : q;
            if (!is_v) raw[j] = (uint16_t)pack16<BF16>(y, 0.0f), raw[j + 4] = (uint16_t)pack16<BF16>(z, 0.0f);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) to[column(j)] = raw[j];
    }
}

// ------------------------------------------------------------------------------------------------ keep
// A thread owns 16 bytes of a head's row in one layer of keys or values and moves them for j = 0, 1, ...: what row j receives
// comes from a row at or behind it (accepted[j] >= j), so no source has been overwritten when it is read, and no thread waits for another.
// Eight sources are requested before the first is written: a source among the eight targets is read first. 64 paths of up to 8 rows in 32
// layers (76 MB): 10.5 to 12 us, by what L2 still holds.
constexpr int kKeepThreads = 256, kKeepSeg = 256, kKeepAhead = 8;

__global__ void __launch_bounds__(kKeepThreads)
    paged_keep_kernel(const PagedView kv, uint4 *kc, uint4 *vc, const int *__restrict__ accepted, int max_accept, const int *__restrict__ count, int *__restrict__ len_out) {
    __shared__ long long from[kKeepSeg], to[kKeepSeg];
    pdl_trigger();
    pdl_wait();
    const int seq = blockIdx.y, len = kv.length(seq), n = min(max(__ldg(count + seq), 0), max_accept);
    if (blockIdx.x == 0 && threadIdx.x == 0) len_out[seq] = len + n;
    const int words = kv.hd / 8;
    const int col = blockIdx.x * kKeepThreads + threadIdx.x, total = kv.layers * 2 * kv.nkv * words;
    const int w = col % words, h = col / words % kv.nkv, lv = col / words / kv.nkv;
    uint4 *base = (lv & 1 ? vc : kc) + (lv >> 1) * (kv.layer_stride / 8) + (long long)h * kv.page * words + w;
    for (int s0 = 0; s0 < n; s0 += kKeepSeg) {
        const int m = min(kKeepSeg, n - s0);
        __syncthreads();
        for (int j = threadIdx.x; j < m; j += kKeepThreads) {
            const int a = __ldg(accepted + (long long)seq * max_accept + s0 + j);
            const long long f = a > s0 + j && a < kv.rows - len ? kv.row_of(seq, len + a) : -1;  // (equal: it lies where it belongs)
            const long long t = f >= 0 ? kv.row_of(seq, len + s0 + j) : -1;
            from[j] = t >= 0 ? f / 8 : -1;
            to[j] = t / 8;
        }
        __syncthreads();
        if (col >= total) continue;
        for (int j = 0; j < m; j += kKeepAhead) {
            uint4 x[kKeepAhead];
#pragma unroll
            for (int i = 0; i < kKeepAhead; i++)
                if (j + i < m && from[j + i] >= 0) x[i] = base[from[j + i]];
#pragma unroll
            for (int i = 0; i < kKeepAhead; i++)
                if (j + i < m && from[j + i] >= 0) base[to[j + i]] = x[i];
        }
    }
}

// ------------------------------------------------------------------------------------------------ reorder
// A block works for one sequence: the first of them writes its table row and length, all copy the rows of its last page where it is not its
// parent's first child. Sources are pages of beams with a child, targets those of beams without (as many as there are further children): no block
// writes what another reads. 32 of 64 beams in 32 layers (150 MB): 27 us, 5.5 TB/s.
constexpr int kReorderThreads = 256, kReorderMost = 256;  // beams of a group: one thread each

__global__ void __launch_bounds__(kReorderThreads)
    paged_reorder_kernel(const PagedView kv, uint4 *kc, uint4 *vc, const int *__restrict__ parent, int group, int *__restrict__ table_out, long long table_out_stride,
                         int *__restrict__ len_out) {
    __shared__ int par[kReorderMost];
    __shared__ int childless[kReorderMost];
    pdl_trigger();
    pdl_wait();
    const int seq = blockIdx.y, g0 = seq / group * group, me = seq - g0, t = threadIdx.x;
    if (t < group) {
        const int p = __ldg(parent + g0 + t);
        par[t] = (unsigned)p < (unsigned)group ? p : t;
        childless[t] = 1;
    }
    __syncthreads();
    if (t < group) childless[par[t]] = 0;
    bool again = false;  // an earlier beam has this one's parent
    if (t < group && t <= me)
        for (int j = 0; j < t; j++) again = again || par[j] == par[t];
    const int nth = __syncthreads_count(again && t < me);  // further children before this one
    const int mine = __syncthreads_or(again && t == me);
    const int src = g0 + par[me], len = kv.length(src), last = len / kv.page, rows = len % kv.page;
    // from index `last` on a further child has the pages that a childless beam has from its own last page on
    int giver = src, shift = 0, own_from = kv.width;
    if (mine) {
        int left = nth, b = 0;
        while (b < group - 1 && !(childless[b] && left-- == 0)) b++;
        giver = g0 + b;
        shift = kv.length(giver) / kv.page - last;
        own_from = last;
    }
    auto entry = [&](int i) {
        if (i < own_from) return __ldg(kv.table + src * kv.table_stride + i);
        return i + shift < kv.width ? __ldg(kv.table + giver * kv.table_stride + i + shift) : -1;
    };
    if (blockIdx.x == 0) {
        for (int i = t; i < kv.width; i += kReorderThreads) table_out[seq * table_out_stride + i] = entry(i);
        if (t == 0) len_out[seq] = len;
    }
    if (!mine || rows == 0 || last >= kv.width) return;
    const int page = entry(last);
    if ((unsigned)page >= (unsigned)kv.pages) return;
    const long long from = kv.page_of(src, len), to = page * kv.page_stride;
    if (from < 0 || from == to) return;
    const int words = kv.hd / 8, span = rows * words;  // 16-byte words of a head: its rows lie in a row
    const int lots = kv.layers * 2 * kv.nkv;
    // a warp takes a head's span in pieces of 32 lanes x 4 words
    const int pieces = (span + 127) / 128;
    const long long total = (long long)lots * pieces;
    for (long long i = (long long)blockIdx.x * (kReorderThreads / 32) + (t >> 5); i < total; i += (long long)gridDim.x * (kReorderThreads / 32)) {
        const int lot = (int)(i / pieces), piece = (int)(i - (long long)lot * pieces);
        const int h = lot % kv.nkv, lv = lot / kv.nkv;
        uint4 *base = (lv & 1 ? vc : kc) + (lv >> 1) * (kv.layer_stride / 8) + (long long)h * kv.page * words;
        uint4 x[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int at = piece * 128 + k * 32 + (t & 31);
            if (at < span) x[k] = base[from / 8 + at];
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int at = piece * 128 + k * 32 + (t & 31);
            if (at < span) base[to / 8 + at] = x[k];
        }
    }
}

}  // namespace
}  // namespace im

// ---- C ABI ------------------------------------------------------------------------------------------------------
namespace im {
namespace {

// What the calls that append have in common: their arguments checked, the kernels' filled in. empty: there is nothing to do.
int append_args(im_device *dev, const im_paged_kv *kv, int layer, const void *k_dev, int64_t k_stride, const void *v_dev, int64_t v_stride, const int *token_start_dev,
                int num_tokens, const void *q_dev, int64_t q_stride, void *q_out_dev, int64_t q_out_stride, int num_heads, const void *cos_dev, const void *sin_dev,
                int table_dtype, int max_pos, int rotary_dim, int neighbours, const int *position_dev, Append *a, bool *empty) {
    *empty = false;
    IM_REQUIRE(layer >= 0, "layer %d", layer);
    int rc = paged_view(kv, layer, &a->kv);
    if (rc != IM_OK) return rc;
    IM_REQUIRE(num_tokens >= 0, "bad argument");
    if (num_tokens == 0 || kv->num_seqs == 0) {
        *empty = true;
        return paged_device(dev);
    }
    IM_REQUIRE(k_dev && v_dev && token_start_dev, "bad argument");
    IM_REQUIRE(!q_dev == !q_out_dev && (q_dev ? num_heads > 0 : num_heads == 0), "queries need their output and number of heads");
    const int64_t row = (int64_t)kv->num_kv_heads * kv->head_dim, q_row = (int64_t)num_heads * kv->head_dim, most = (int64_t)1 << 40;
    IM_REQUIRE(k_stride >= row && v_stride >= row && k_stride <= most && v_stride <= most && k_stride % 8 == 0 && v_stride % 8 == 0 && aligned16(k_dev) && aligned16(v_dev),
               "rows of keys and values have to be 16-byte aligned and apart");
    IM_REQUIRE(!q_dev || (q_stride >= q_row && q_out_stride >= q_row && q_stride <= most && q_out_stride <= most && q_stride % 8 == 0 && q_out_stride % 8 == 0 &&
                          aligned16(q_dev) && aligned16(q_out_dev)),
               "rows of queries have to be 16-byte aligned and apart");
    IM_REQUIRE(num_heads <= kAppendMost && kv->num_kv_heads <= kAppendMost, "%d and %d heads (at most %d)", num_heads, kv->num_kv_heads, kAppendMost);
    IM_REQUIRE(!q_dev || (q_out_dev == q_dev && (q_out_stride == q_stride || num_tokens == 1)) || !share_rows(q_dev, 2 * q_stride, q_out_dev, 2 * q_out_stride, 2 * q_row, num_tokens),
               "the rotated queries lie over other tokens' queries");
    IM_REQUIRE(rotary_dim >= 0 && rotary_dim <= kv->head_dim && rotary_dim % 2 == 0, "rotary_dim %d of %d", rotary_dim, kv->head_dim);
    IM_REQUIRE(rotary_dim == 0 || (cos_dev && sin_dev && max_pos > 0 && (table_dtype == IM_DTYPE_F16 || table_dtype == IM_DTYPE_F32)),
               "rotation needs tables of cosines and sines in fp16 or f32");
    IM_REQUIRE(rotary_dim == 0 || (aligned16(cos_dev) && aligned16(sin_dev)), "tables of cosines and sines have to be 16-byte aligned");
    IM_REQUIRE(neighbours == 0 || neighbours == 1, "neighbours is 0 or 1");
    rc = paged_device(dev);
    if (rc != IM_OK) return rc;
    const int64_t at = layer * (int64_t)a->kv.layer_stride;
    a->kc = static_cast<uint16_t *>(kv->k_dev) + at;
    a->vc = static_cast<uint16_t *>(kv->v_dev) + at;
    a->k = static_cast<const uint16_t *>(k_dev);
    a->v = static_cast<const uint16_t *>(v_dev);
    a->q = static_cast<const uint16_t *>(q_dev);
    a->qo = static_cast<uint16_t *>(q_out_dev);
    a->ks = k_stride; a->vs = v_stride; a->qs = q_stride; a->qos = q_out_stride;
    a->start = token_start_dev; a->pos = position_dev;
    a->cosc = cos_dev; a->sinc = sin_dev;
    a->nh = num_heads; a->max_pos = max_pos; a->rot = rotary_dim;
    return IM_OK;
}

// Lanes that hold a head.
int append_lanes(int head_dim) {
    int lanes = 1;
    while (lanes * 8 < head_dim) lanes *= 2;
    return lanes;
}

}  // namespace
}  // namespace im

IM_EXPORT int im_cuda_paged_append(im_device *dev, const im_paged_kv *kv, int layer, const void *k_dev, int64_t k_stride, const void *v_dev, int64_t v_stride,
                                   const int *token_start_dev, int num_tokens, const void *q_dev, int64_t q_stride, void *q_out_dev, int64_t q_out_stride,
                                   int num_heads, const void *cos_dev, const void *sin_dev, int table_dtype, int max_pos, int rotary_dim, int neighbours,
                                   const int *position_dev, void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    Append a;
    bool empty;
    const int rc = append_args(dev, kv, layer, k_dev, k_stride, v_dev, v_stride, token_start_dev, num_tokens, q_dev, q_stride, q_out_dev, q_out_stride, num_heads, cos_dev, sin_dev,
                               table_dtype, max_pos, rotary_dim, neighbours, position_dev, &a, &empty);
    if (rc != IM_OK || empty) return rc;
    const int lanes = append_lanes(kv->head_dim);
    const bool bf16 = kv->dtype == IM_DTYPE_BF16, f32 = table_dtype == IM_DTYPE_F32;
    const int form = rotary_dim == 0 ? 0 : neighbours ? 2 : rotary_dim % 16 == 0 ? 1 : 3;
    void (*kern)(Append, int) = nullptr;
#define IM_FORM(F) (bf16 ? (f32 ? paged_append_kernel<true, F, true> : paged_append_kernel<true, F, false>) : (f32 ? paged_append_kernel<false, F, true> : paged_append_kernel<false, F, false>))
    switch (form) {
    case 0: kern = bf16 ? paged_append_kernel<true, 0, false> : paged_append_kernel<false, 0, false>; break;
    case 1: kern = IM_FORM(1); break;
    case 2: kern = IM_FORM(2); break;
    default: kern = IM_FORM(3); break;
    }
#undef IM_FORM
    IM_CUDA_CHECK(launch_k(kern, dim3((unsigned)num_tokens), dim3(num_tokens > 4 * dev->sm_count ? kAppendSmall : kAppendThreads), 0, as_stream(stream), a, lanes));
    return IM_OK;
    IM_GUARD_END
}

IM_EXPORT int im_cuda_paged_append_normed(im_device *dev, const im_paged_kv *kv, const im_paged_append_args *args, void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    IM_REQUIRE(kv && args, "kv or args is NULL");
    const im_paged_append_args &x = *args;
    IM_REQUIRE(!x.q_norm_dev || x.num_heads > 0, "norm weights of queries without queries");
    IM_REQUIRE((!x.q_norm_dev && !x.k_norm_dev) || x.norm_dtype == IM_DTYPE_F32 || x.norm_dtype == kv->dtype, "norm weights are of the cache's type or f32 (got dtype %d)", x.norm_dtype);
    IM_REQUIRE(aligned16(x.q_norm_dev) && aligned16(x.k_norm_dev), "norm weights have to be 16-byte aligned");
    IM_REQUIRE(x.eps >= 0.0f && x.eps - x.eps == 0.0f, "eps has to be finite and not negative");
    IM_REQUIRE(x.num_axes >= 1 && x.num_axes <= kAxes, "%d axes (at most %d)", x.num_axes, kAxes);
    IM_REQUIRE(x.num_axes == 1 || (x.rotary_dim > 0 && (x.position_dev || x.num_tokens == 0) && x.pair_axis_host), "several axes need a rotation, positions and the axis of every pair");
    Append a;
    bool empty;
    const int rc = append_args(dev, kv, x.layer, x.k_dev, x.k_stride, x.v_dev, x.v_stride, x.token_start_dev, x.num_tokens, x.q_dev, x.q_stride, x.q_out_dev, x.q_out_stride, x.num_heads,
                               x.cos_dev, x.sin_dev, x.table_dtype, x.max_pos, x.rotary_dim, x.neighbours, x.position_dev, &a, &empty);
    if (rc != IM_OK || empty) return rc;
    AppendMore m{};
    m.qn = x.q_norm_dev; m.kn = x.k_norm_dev;
    m.norm_f32 = x.norm_dtype == IM_DTYPE_F32;
    m.axes = x.num_axes;
    m.neighbours = x.neighbours;
    m.eps = x.eps;
    m.inv_dim = 1.0f / kv->head_dim;
    for (int i = 0; x.num_axes > 1 && i < x.rotary_dim / 2; i++) {
        IM_REQUIRE(x.pair_axis_host[i] < x.num_axes, "pair %d on axis %d of %d", i, x.pair_axis_host[i], x.num_axes);
        m.axis[i / 16] |= (uint32_t)x.pair_axis_host[i] << (2 * (i % 16));
    }
    const int lanes = append_lanes(kv->head_dim);
    const bool bf16 = kv->dtype == IM_DTYPE_BF16, f32 = x.table_dtype == IM_DTYPE_F32;
    const dim3 grid((unsigned)x.num_tokens), block(x.num_tokens > 4 * dev->sm_count ? kAppendSmall : kAppendThreads);
    if (x.rotary_dim % 8) {
        void (*odd)(Append, AppendMore, int) = bf16 ? (f32 ? paged_append_odd_kernel<true, true> : paged_append_odd_kernel<true, false>)
                                                    : (f32 ? paged_append_odd_kernel<false, true> : paged_append_odd_kernel<false, false>);
        IM_CUDA_CHECK(launch_k(odd, grid, block, 0, as_stream(stream), a, m, lanes));
        return IM_OK;
    }
    void (*kern)(Append, AppendMore) = nullptr;
#define IM_LANES(B, N, F) (lanes == 32 ? paged_append_normed_kernel<B, N, F, 32> : lanes == 16 ? paged_append_normed_kernel<B, N, F, 16> : paged_append_normed_kernel<B, N, F, 8>)
#define IM_FORM(B, F) (x.neighbours ? IM_LANES(B, true, F) : IM_LANES(B, false, F))
    kern = bf16 ? (f32 ? IM_FORM(true, true) : IM_FORM(true, false)) : (f32 ? IM_FORM(false, true) : IM_FORM(false, false));
#undef IM_FORM
#undef IM_LANES
    IM_CUDA_CHECK(launch_k(kern, grid, block, 0, as_stream(stream), a, m));
    return IM_OK;
    IM_GUARD_END
}

IM_EXPORT int im_cuda_paged_keep(im_device *dev, const im_paged_kv *kv, const int *accepted_dev, int max_accept, const int *count_dev, int *seq_len_out_dev,
                                 void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    PagedView v;
    int rc = paged_view(kv, -1, &v);
    if (rc != IM_OK) return rc;
    IM_REQUIRE(max_accept >= 1 && (v.nseq == 0 || (accepted_dev && count_dev && seq_len_out_dev)), "bad argument");
    IM_REQUIRE(kv->num_seqs <= 65535, "at most 65535 sequences (got %d)", kv->num_seqs);
    IM_REQUIRE(!share_memory(seq_len_out_dev, 4ll * v.nseq, v.len, 4ll * v.nseq), "the new lengths lie over the old ones");
    IM_REQUIRE(!share_memory(seq_len_out_dev, 4ll * v.nseq, count_dev, 4ll * v.nseq) && !share_memory(seq_len_out_dev, 4ll * v.nseq, accepted_dev, 4ll * v.nseq * max_accept),
               "the new lengths lie over the accepted places");
    IM_REQUIRE(v.nseq == 0 || !share_memory(seq_len_out_dev, 4ll * v.nseq, v.table, 4 * ((v.nseq - 1) * v.table_stride + v.width)), "the new lengths lie over the page table");
    const long long cols = (long long)v.layers * 2 * v.nkv * (v.hd / 8);
    IM_REQUIRE(cols <= INT_MAX - kKeepThreads, "too many layers and heads");
    rc = paged_device(dev);
    if (rc != IM_OK) return rc;
    if (v.nseq == 0) return IM_OK;
    IM_CUDA_CHECK(launch_k(paged_keep_kernel, dim3((unsigned)((cols + kKeepThreads - 1) / kKeepThreads), v.nseq), dim3(kKeepThreads), 0, as_stream(stream), v,
                           static_cast<uint4 *>(kv->k_dev), static_cast<uint4 *>(kv->v_dev), accepted_dev, max_accept, count_dev, seq_len_out_dev));
    return IM_OK;
    IM_GUARD_END
}

IM_EXPORT int im_cuda_paged_reorder(im_device *dev, const im_paged_kv *kv, const int *parent_dev, int group, int *table_out_dev, int64_t table_out_stride,
                                    int *seq_len_out_dev, void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    PagedView v;
    int rc = paged_view(kv, -1, &v);
    if (rc != IM_OK) return rc;
    IM_REQUIRE(v.nseq == 0 || (parent_dev && table_out_dev && seq_len_out_dev), "bad argument");
    IM_REQUIRE(group >= 1 && group <= kReorderMost && kv->num_seqs % group == 0, "%d sequences in groups of %d (at most %d)", kv->num_seqs, group, kReorderMost);
    IM_REQUIRE(kv->num_seqs <= 65535, "at most 65535 sequences (got %d)", kv->num_seqs);
    const int64_t stride = table_out_stride ? table_out_stride : v.width;
    IM_REQUIRE(stride >= v.width, "rows of the new page table overlap");
    if (v.nseq > 0) {
        const long long lens = 4ll * v.nseq, old_n = 4 * ((v.nseq - 1) * v.table_stride + v.width), new_n = 4 * ((v.nseq - 1) * stride + v.width);
        IM_REQUIRE(!share_memory(table_out_dev, new_n, v.table, old_n) && !share_memory(table_out_dev, new_n, v.len, lens), "the new page table lies over the old one or the lengths");
        IM_REQUIRE(!share_memory(seq_len_out_dev, lens, v.len, lens) && !share_memory(seq_len_out_dev, lens, v.table, old_n),
                   "the new lengths lie over the old ones or the page table");
        IM_REQUIRE(!share_memory(table_out_dev, new_n, parent_dev, lens) && !share_memory(seq_len_out_dev, lens, parent_dev, lens) &&
                       !share_memory(table_out_dev, new_n, seq_len_out_dev, lens),
                   "the new page table and lengths lie over the parents or each other");
    }
    rc = paged_device(dev);
    if (rc != IM_OK) return rc;
    if (v.nseq == 0) return IM_OK;
    // Blocks of a sequence: four pieces for every warp of a full last page, no more than about eight waves over the GPU
    const long long pieces = (long long)v.layers * 2 * v.nkv * (((long long)v.page * (v.hd / 8) + 127) / 128);
    const long long by_work = (pieces + 31) / 32, by_gpu = (64ll * dev->sm_count + v.nseq - 1) / v.nseq;
    const unsigned blocks = (unsigned)std::max(1ll, std::min(by_work, by_gpu));
    IM_CUDA_CHECK(launch_k(paged_reorder_kernel, dim3(blocks, v.nseq), dim3(kReorderThreads), 0, as_stream(stream), v, static_cast<uint4 *>(kv->k_dev),
                           static_cast<uint4 *>(kv->v_dev), parent_dev, group, table_out_dev, (long long)stride, seq_len_out_dev));
    return IM_OK;
    IM_GUARD_END
}
