// The best continuations of a group of beams: value[b, v] = score[b] + x[b, v] - lse[b], lse[b] = log sum_v exp(x[b, v]), the `picks` largest over
// beams and vocabulary, ties to the lowest b * V + v.
//
// The logits are read once, from HBM; what bounds the pass is that read. Within a beam the order of the values is the order of its
// logits, so nothing needs lse before the end: a block walks a slice of a row once for both the running maximum and sum of
// exponentials and the slice's best `picks` logits, and a block per group joins the slices.
//   best of a slice   each thread knows the maximum of what it has met; the picks-th largest of the maxima of 64 sets of threads is a bound that at
//                     least `picks` elements reach. It is taken after the
//                     first, third, ninth and every 32nd piece of the slice and after the last; few elements that do not belong to the best reach it. A
//                     thread only notes which sixteen elements of a piece reach the bound; those that reach the last one are read again and collected.
//                     A collected element's rank is the number of better ones. Where a list overflows (ties, rising rows) the elements are picked one
//                     after the other from memory instead.
//   joining           the same with the slices' picks as elements and 64-bit values.
// Eight beams of 32 searches over 128256 f32 logits, 16 picks (131 MB): 32 us, of them 28 for the slices (4.7 TB/s, 72 % of a copy).
// Sums are f32 per thread over its elements with one running maximum, joined in a fixed order: a run repeats bit by bit. Which elements are a thread's
// goes by their place in the row alone, wherever the row starts: equal rows get equal sums, and their candidates tie as they should.
#include <cuda_bf16.h>
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "cluster.cuh"
#include "paged.cuh"

namespace im {
namespace {

constexpr int kSelThreads = 256, kSelMost = 64, kSelBuf = 1024;
constexpr int kSelResident = 7;  // blocks of an SM
constexpr int kSelLeast = 2048;  // elements of a slice: one request of 16-bit logits for every thread

struct Select {
    const void *x;
    long long stride;
    int groups, beams, vocab, picks, slices, slice;  // slice: elements, a multiple of eight
    const float *score;
    const uint8_t *done;
    int end_token;
    float *score_out;
    int *parent_out, *token_out;
    float *part_v;  // [rows, slices, picks]
    int *part_i;
    float2 *part_ms;  // [rows, slices]: maximum, sum of exp(x - maximum)
};

template <int DT>
struct Logit;
template <>
struct Logit<IM_DTYPE_F32> {
    using T = float;
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ void split(const uint4 &u, float *o) {
        o[0] = __uint_as_float(u.x); o[1] = __uint_as_float(u.y); o[2] = __uint_as_float(u.z); o[3] = __uint_as_float(u.w);
    }
};
template <bool BF16>
struct Logit16 {
    using T = uint16_t;
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float get(uint16_t v) { return BF16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v)); }
    static __device__ __forceinline__ void split(const uint4 &u, float *o) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 t = unpack16<BF16>(w[i]);
            o[2 * i] = t.x;
            o[2 * i + 1] = t.y;
        }
    }
};
template <>
struct Logit<IM_DTYPE_F16> : Logit16<false> {};
template <>
struct Logit<IM_DTYPE_BF16> : Logit16<true> {};

// Larger values first, then lower indexes.
__device__ __forceinline__ bool before(double a, long long ia, double b, long long ib) { return a > b || (a == b && ia < ib); }
__device__ __forceinline__ bool before(float a, int ia, float b, int ib) { return a > b || (a == b && ia < ib); }

// exp(x), zero where it would be denormal
__device__ __forceinline__ float exp_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

// What reaches the bound, and the best of it.
template <typename V, typename I, int BUF>
struct Best {
    V buf_v[BUF];
    I buf_i[BUF];
    V out_v[kSelMost];
    I out_i[kSelMost];
    V tops[kSelThreads], low;
    int count;

    __device__ __forceinline__ void clear(int picks) {  // no synchronisation: the first bound() has one
        if (threadIdx.x == 0) count = 0;
        for (int i = threadIdx.x; i < picks; i += kSelThreads) out_v[i] = -INFINITY, out_i[i] = -1;
    }
    // The picks-th largest of the maxima of 64 sets of threads; top: this thread's maximum so far. A set has every 64th thread, so that none is without
    // elements where the first threads have some. (Of random elements ln 2 a set reach the bound for 32 picks, 1 / 4 for 16.)
    __device__ __forceinline__ V bound(V top, int picks) {
        __syncthreads();
        tops[threadIdx.x] = top;
        __syncthreads();
        if (threadIdx.x < 32) {
            V a = tops[threadIdx.x], b = tops[32 + threadIdx.x];
#pragma unroll
            for (int w = 2; w < kSelThreads / 32; w += 2) {
                const V x = tops[32 * w + threadIdx.x], y = tops[32 * w + 32 + threadIdx.x];
                a = a > x ? a : x;
                b = b > y ? b : y;
            }
            int above_a = 0, above_b = 0;
#pragma unroll 8
            for (int j = 0; j < 32; j++) {
                const V x = __shfl_sync(0xffffffffu, a, j), y = __shfl_sync(0xffffffffu, b, j);
                above_a += (x > a) + (y > a);
                above_b += (x > b) + (y > b);
            }
            V v = INFINITY;  // the lowest of those with fewer than `picks` above
            if (above_a < picks) v = a;
            if (above_b < picks) v = v < b ? v : b;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const V x = __shfl_xor_sync(0xffffffffu, v, o);
                v = v < x ? v : x;
            }
            if (threadIdx.x == 0) low = v;
        }
        __syncthreads();
        return low;
    }
    __device__ __forceinline__ void collect(V v, I i) {
        const int at = atomicAdd(&count, 1);
        if (at < BUF) buf_v[at] = v, buf_i[at] = i;
    }
    // The best into out_v, out_i, in order. visit(f) hands all elements of this thread to f(value, index).
    template <typename Visit>
    __device__ __forceinline__ void rank(int picks, Visit visit) {
        __syncthreads();
        const int t = threadIdx.x, n = count;
        if (n <= BUF) {
            for (int i = t; i < n; i += kSelThreads) {
                const V v = buf_v[i];
                const I x = buf_i[i];
                int r = 0;
                for (int j = 0; j < n; j++) r += before(buf_v[j], buf_i[j], v, x);
                if (r < picks) out_v[r] = v, out_i[r] = x;
            }
        } else {
            V last_v = INFINITY;
            I last_i = -1;
            for (int k = 0; k < picks; k++) {
                V v = -INFINITY;
                I x = 0x7fffffff;
                visit([&](V value, I index) {
                    if (value > -INFINITY && before(last_v, last_i, value, index) && (before(value, index, v, x) || !(v > -INFINITY))) v = value, x = index;
                });
#pragma unroll 1
                for (int o = 16; o > 0; o >>= 1) {
                    const V v2 = __shfl_xor_sync(0xffffffffu, v, o);
                    const I x2 = __shfl_xor_sync(0xffffffffu, x, o);
                    if (before(v2, x2, v, x)) v = v2, x = x2;
                }
                __syncthreads();
                if ((t & 31) == 0) buf_v[t >> 5] = v, buf_i[t >> 5] = x;
                __syncthreads();
                v = buf_v[0], x = buf_i[0];
                for (int w = 1; w < kSelThreads / 32; w++)
                    if (before(buf_v[w], buf_i[w], v, x)) v = buf_v[w], x = buf_i[w];
                if (!(v > -INFINITY)) break;
                if (t == 0) out_v[k] = v, out_i[k] = x;
                last_v = v;
                last_i = x;
            }
        }
        __syncthreads();
    }
};

// A slice of a row: its best logits in order in best.out_v / out_i, its maximum and sum of exponentials.
struct SliceSpace {
    Best<float, int, kSelBuf> best;
    float red_m[kSelThreads / 32], red_s[kSelThreads / 32];
    float met_v[kSelBuf];  // sixteen elements of a thread that reach the bound: their maximum, and which
    int met_i[kSelBuf], kept[kSelBuf], met, keep;
    float2 ms;
};

// ANY: some row does not start at a multiple of 16 bytes. Elements are read one by one then, 32 of a warp side by side, from all rows (32 x 8 beams
// over 128257 f32 logits 36 us, 128256 32; 16-bit ones 31 and 29; shifting aligned pieces into place cost more, 36 and 33).
template <int DT, bool ANY>
__device__ __forceinline__ void slice_best(const Select &p, long long row, int slice, SliceSpace &sp) {
    using L = Logit<DT>;
    using T = typename L::T;
    constexpr int V = L::kVec, Q = 16 / V;  // requests of a piece: 16 elements of each thread
    constexpr int kPiece = (ANY ? 16 : Q) * kSelThreads;
    auto &best = sp.best;
    auto &met = sp.met;
    auto &keep = sp.keep;
    float *red_m = sp.red_m, *red_s = sp.red_s, *met_v = sp.met_v;
    int *met_i = sp.met_i, *kept = sp.kept;
    const int t = threadIdx.x;
    const T *x = static_cast<const T *>(p.x) + row * p.stride;
    const int a = slice * p.slice, b = min(a + p.slice, p.vocab);
    // 16 bytes of elements at a time from the first one on (a is a multiple of eight elements); what is left behind them is read one by one
    const int vecs = max(b - a, 0) / V, tail = ANY ? b : a + vecs * V;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + a);
    best.clear(p.picks);
    if (t == 0) met = keep = 0;
    float m = -INFINITY, s = 0.0f;
    // running maximum and sum; (x - m) first: it is exact where it matters, a product with log2(e) is not
    auto take = [&](const float *f, int n, float top) {
        if (top > m) {
            s *= exp_of(m - top);
            m = top;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int j = 0; j < n; j += 2) {
            a += exp_of(f[j] - base);
            if (j + 1 < n) b += exp_of(f[j + 1] - base);
        }
        s += a + b;
    };
    // the odd end: up to 7 elements, the first threads' (with no bound yet: collected where they reach the first one)
    const int ends = max(b - tail, 0), end_at = tail + t;
    float end = -INFINITY;
    if (t < ends) {
        end = L::get(x[end_at]);
        take(&end, 1, end);
    }
    const int pieces = (max(b - a, 0) / (ANY ? 1 : V) + kPiece - 1) / kPiece;
    float bound = -INFINITY;
#pragma unroll 1
    for (int k = 0; k < max(pieces, 1); k++) {
        const int i0 = ANY ? a + k * kPiece + (t & ~31) * 16 + (t & 31) : k * kPiece + t;
        float f[16];
        if constexpr (ANY) {
            T e[16];
            if (i0 + 15 * 32 < b) {
#pragma unroll
                for (int j = 0; j < 16; j++) e[j] = __ldg(x + i0 + j * 32);
#pragma unroll
                for (int j = 0; j < 16; j++) f[j] = L::get(e[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 16; j++) f[j] = i0 + j * 32 < b ? L::get(__ldg(x + i0 + j * 32)) : -INFINITY;
            }
        } else if (i0 + (Q - 1) * kSelThreads < vecs) {
            uint4 u[Q];
#pragma unroll
            for (int q = 0; q < Q; q++) u[q] = ldg_stream_v4(xv + i0 + q * kSelThreads);
#pragma unroll
            for (int q = 0; q < Q; q++) L::split(u[q], f + q * V);
        } else {
#pragma unroll
            for (int q = 0; q < Q; q++) {
                const bool in = i0 + q * kSelThreads < vecs;
                uint4 u = make_uint4(0, 0, 0, 0);
                if (in) u = ldg_stream_v4(xv + i0 + q * kSelThreads);
                L::split(u, f + q * V);
                if (!in)
#pragma unroll
                    for (int j = 0; j < V; j++) f[q * V + j] = -INFINITY;
            }
        }
        float top4[4];
#pragma unroll
        for (int j = 0; j < 4; j++) top4[j] = fmaxf(fmaxf(f[4 * j], f[4 * j + 1]), fmaxf(f[4 * j + 2], f[4 * j + 3]));
        const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
        take(f, 16, top);
        if (k == 0 || k == 2 || k == 8 || (k & 31) == 31) bound = best.bound(m, p.picks);
        if (top >= bound && top > -INFINITY) {
            const int at = atomicAdd(&met, 1);
            if (at < kSelBuf) met_v[at] = top, met_i[at] = i0;
        }
    }
    if (pieces > 1) bound = best.bound(m, p.picks);
    else __syncthreads();
    const int n = met;
    if (n <= kSelBuf) {
        for (int i = t; i < n; i += kSelThreads)
            if (met_v[i] >= bound) kept[atomicAdd(&keep, 1)] = met_i[i];
        __syncthreads();
        for (int i = t; i < keep * 16; i += kSelThreads) {
            const int at = kept[i >> 4], v = at + (i & 15) / V * kSelThreads, e = ANY ? at + (i & 15) * 32 : a + v * V + (i & 15) % V;
            if (ANY ? e >= b : v >= vecs) continue;
            const float f = L::get(x[e]);
            if (f >= bound && f > -INFINITY) best.collect(f, e);
        }
        if (end >= bound && end > -INFINITY) best.collect(end, end_at);
    } else if (t == 0) {
        best.count = INT_MAX;  // too many: one after the other
    }
    // joined over lanes, then warps, in a fixed order
    float M = warp_max(m);
    float S = warp_sum(m == -INFINITY && s == 0.0f ? 0.0f : s * exp_of(m - M));
    if ((t & 31) == 0) red_m[t >> 5] = M, red_s[t >> 5] = S;
    best.rank(p.picks, [&](auto f) {
        if (t < ends) f(end, end_at);
        if constexpr (ANY) {
            for (int e = a + t; e < b; e += kSelThreads) f(L::get(x[e]), e);
        } else {
            for (int i = t; i < vecs; i += kSelThreads) {
                float g[V];
                L::split(__ldg(xv + i), g);
                for (int j = 0; j < V; j++) f(g[j], a + i * V + j);
            }
        }
    });
    if (t == 0) {
        M = -INFINITY;
        for (int w = 0; w < kSelThreads / 32; w++) M = fmaxf(M, red_m[w]);
        S = 0.0f;
        for (int w = 0; w < kSelThreads / 32; w++) S += red_m[w] == -INFINITY && red_s[w] == 0.0f ? 0.0f : red_s[w] * exp_of(red_m[w] - M);
        sp.ms = make_float2(M, S);
    }
    __syncthreads();
}

// grid (slices, rows)
template <int DT, bool ANY>
__global__ void __launch_bounds__(kSelThreads, kSelResident) beam_slice_kernel(const __grid_constant__ Select p) {
    __shared__ SliceSpace sp;
    pdl_trigger();
    pdl_wait();
    const int slice = blockIdx.x, t = threadIdx.x;
    const long long row = blockIdx.y;
    if (p.done && p.done[row]) return;
    slice_best<DT, ANY>(p, row, slice, sp);
    if (t == 0) p.part_ms[row * p.slices + slice] = sp.ms;
    const long long at = (row * p.slices + slice) * p.picks;
    for (int k = t; k < p.picks; k += kSelThreads) {
        p.part_v[at + k] = sp.best.out_v[k];
        p.part_i[at + k] = sp.best.out_i[k];
    }
}

// What the slices of a group's beams found, joined.
constexpr int kHeld = 4 * kSelThreads;  // candidates that fit shared memory
struct JoinSpace {
    Best<double, long long, kSelBuf / 2> best;
    double offset[kSelMost];  // score - lse of each beam; NaN: nothing of it is picked
    float held_v[kHeld];
    int held_i[kHeld];
};

// ms: maxima and sums of the beams' slices; held: all candidates (on their way, where they come from memory) are in held_v, held_i
__device__ __forceinline__ void join_group(const Select &p, int group, const float2 *ms, bool held, JoinSpace &sp) {
    auto &best = sp.best;
    double *offset = sp.offset;
    const int t = threadIdx.x, lane = t & 31;
    const long long row0 = (long long)group * p.beams;
    const int per = p.slices * p.picks, n = p.beams * per;
    best.clear(p.picks);
    for (int b = t >> 5; b < p.beams; b += kSelThreads / 32) {
        const bool done = p.done && p.done[row0 + b];
        float m = -INFINITY, s = 0.0f;
        if (!done) {
            const float2 none = make_float2(-INFINITY, 0.0f), x = lane < p.slices ? ms[b * p.slices + lane] : none, y = lane + 32 < p.slices ? ms[b * p.slices + lane + 32] : none;
            m = warp_max(fmaxf(x.x, y.x));
            if (!(x.x == -INFINITY && x.y == 0.0f)) s += x.y * expf(x.x - m);
            if (!(y.x == -INFINITY && y.y == 0.0f)) s += y.y * expf(y.x - m);
            s = warp_sum(s);
        }
        if (lane == 0) {
            const double lse = (double)m + log((double)s);
            offset[b] = done ? (double)p.score[row0 + b] : lse > -INFINITY && lse < INFINITY ? (double)p.score[row0 + b] - lse : NAN;
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    auto visit = [&](auto f) {  // an index is (beam, token)
#pragma unroll 1
        for (int i = t; i < n; i += kSelThreads) {
            const float v = held ? sp.held_v[i] : p.part_v[row0 * per + i];
            const int token = held ? sp.held_i[i] : p.part_i[row0 * per + i], b = i / per, k = i - b * per;
            if (p.done && p.done[row0 + b]) {
                if (k == 0) f(offset[b], (long long)b << 32 | p.end_token);
            } else if (token >= 0) {
                f(offset[b] + (double)v, (long long)b << 32 | token);
            }
        }
    };
    double top = -INFINITY;
    visit([&](double value, long long) { if (value > top) top = value; });
    const double bound = best.bound(top, p.picks);
    if (top >= bound && top > -INFINITY)
        visit([&](double value, long long index) { if (value >= bound && value > -INFINITY) best.collect(value, index); });
    best.rank(p.picks, visit);
    for (int k = t; k < p.picks; k += kSelThreads) {
        const long long i = best.out_i[k], at = (long long)group * p.picks + k;
        p.score_out[at] = (float)best.out_v[k];
        p.parent_out[at] = i < 0 ? -1 : (int)(i >> 32);
        p.token_out[at] = i < 0 ? -1 : (int)i;
    }
}

// grid (groups)
__global__ void __launch_bounds__(kSelThreads) beam_join_kernel(const __grid_constant__ Select p) {
    __shared__ JoinSpace sp;
    pdl_trigger();
    pdl_wait();
    const int per = p.slices * p.picks, n = p.beams * per;
    const long long row0 = (long long)blockIdx.x * p.beams;
    if (n <= kHeld) {  // on its way while lse is computed
        for (int i = threadIdx.x; i < n; i += kSelThreads) {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(sp.held_v + i)), "l"(p.part_v + row0 * per + i) : "memory");
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(sp.held_i + i)), "l"(p.part_i + row0 * per + i) : "memory");
        }
    }
    join_group(p, blockIdx.x, p.part_ms + row0 * p.slices, n <= kHeld, sp);
}

// Few beams over few elements: a cluster per group, a CTA per slice of a beam; the first one joins what it finds in the others' shared memory. One
// launch, no scratch: the host's part of a call is what there is to save (four beams over 32768: 12.6 us a call from Python, 17.8 in two launches). On the
// device two launches are the shorter ones, 7.2 us against 10.0 in a captured graph, and the more so the longer the slices (four beams: of 65536 7.8 and
// 12.0, of 128256 9.4 and 21.4) and the fewer the clusters that the GPU holds leave free (40 searches of four beams 13.8 and 15.5): the limits.
constexpr int kSelCluster = 8, kSelClusterSlice = 32768;
template <int DT, bool ANY>
__global__ void __launch_bounds__(kSelThreads) beam_cluster_kernel(const __grid_constant__ Select p) {
    __shared__ SliceSpace sp;
    __shared__ JoinSpace js;
    __shared__ float2 ms[kSelCluster];
    pdl_trigger();
    pdl_wait();
    const int C = p.beams * p.slices, group = blockIdx.x / C, rank = blockIdx.x - group * C, beam = rank / p.slices;
    const long long row = (long long)group * p.beams + beam;
    if (!(p.done && p.done[row])) slice_best<DT, ANY>(p, row, rank - beam * p.slices, sp);
    cluster_sync();
    if (rank == 0) {
        for (int i = threadIdx.x; i < C * p.picks; i += kSelThreads) {  // (what a finished beam's CTA holds is not looked at)
            const int from = i / p.picks, k = i - from * p.picks;
            js.held_v[i] = __uint_as_float(remote1(of_rank(sp.best.out_v + k, from)));
            js.held_i[i] = (int)remote1(of_rank(sp.best.out_i + k, from));
        }
        if (threadIdx.x < C) ms[threadIdx.x] = remote2(of_rank(&sp.ms, threadIdx.x));
        __syncthreads();
    }
    cluster_sync();  // nobody leaves while another reads what it has
    if (rank == 0) join_group(p, group, ms, true, js);
}

// Slices of a beam where a cluster takes a group, 0 where it does not.
int cluster_slices(const Device *dev, int groups, int beams, int vocab) {
    if (beams > kSelCluster) return 0;
    const int n = std::max(1, std::min(kSelCluster / beams, (vocab + kSelLeast - 1) / kSelLeast));
    return (vocab + n - 1) / n <= kSelClusterSlice && (long long)groups * beams * n <= 2ll * dev->sm_count ? n : 0;
}
// Slices of a row: as many as the GPU holds blocks of all rows at a time (a second wave of a few would cost as much as a full one), none below kSelLeast
// elements.
int select_slices(const Device *dev, int groups, int beams, int vocab) {
    const long long rows = (long long)groups * beams;
    const long long want = (long long)kSelResident * dev->sm_count / rows, most = (vocab + kSelLeast - 1) / kSelLeast;
    return (int)std::max(1ll, std::min(std::min(want, most), 64ll));
}
size_t select_bytes(long long rows, int slices, int picks) { return (size_t)rows * slices * (8 + 8 * (size_t)picks) + 16; }

}  // namespace
}  // namespace im

IM_EXPORT size_t im_cuda_beam_select_scratch_bytes(const im_device *dev, int groups, int beams, int vocab, int picks) {
    if (dev && groups >= 1 && beams >= 1 && vocab >= 1 && im::cluster_slices(dev, groups, beams, vocab)) return 0;
    if (!dev || groups < 1 || beams < 1 || beams > im::kSelMost || vocab < 1 || picks < 1 || picks > im::kSelMost || (long long)groups * beams > 65535) return 0;
    return im::select_bytes((long long)groups * beams, im::select_slices(dev, groups, beams, vocab), picks);
}

IM_EXPORT int im_cuda_beam_select(im_device *dev, const void *logits_dev, int dtype, int64_t row_stride, int groups, int beams, int vocab, const float *score_dev,
                                  const uint8_t *done_dev, int end_token, int picks, float *score_out_dev, int *parent_out_dev, int *token_out_dev,
                                  void *scratch_dev, size_t scratch_bytes, void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    IM_REQUIRE(dtype == IM_DTYPE_F16 || dtype == IM_DTYPE_F32 || dtype == IM_DTYPE_BF16, "logits are fp16, bf16 or f32 (got dtype %d)", dtype);
    IM_REQUIRE(groups >= 0 && beams >= 1 && beams <= kSelMost && vocab >= 1 && vocab <= INT_MAX - 65536, "%d groups of %d beams (at most %d) over %d tokens", groups, beams, kSelMost, vocab);
    IM_REQUIRE(picks >= 1 && picks <= kSelMost, "1 to %d picks (got %d)", kSelMost, picks);
    IM_REQUIRE((long long)groups * beams <= 65535, "at most 65535 beams in all (got %lld)", (long long)groups * beams);
    IM_REQUIRE(row_stride == 0 || (row_stride >= vocab && row_stride <= (int64_t)1 << 40), "rows of logits overlap");
    IM_REQUIRE(groups == 0 || (logits_dev && score_dev && score_out_dev && parent_out_dev && token_out_dev), "a pointer is NULL");
    IM_REQUIRE(!share_memory(score_out_dev, 4ll * groups * picks, score_dev, 4ll * groups * beams), "the new scores lie over the old ones");
    IM_REQUIRE(reinterpret_cast<uintptr_t>(logits_dev) % (dtype == IM_DTYPE_F32 ? 4 : 2) == 0, "logits are not aligned to their type");
    IM_REQUIRE(!done_dev || (end_token >= 0 && end_token < vocab), "end_token %d of %d", end_token, vocab);
    int rc = paged_device(dev);
    if (rc != IM_OK) return rc;
    if (groups == 0) return IM_OK;
    Select p;
    const int clustered = cluster_slices(dev, groups, beams, vocab);
    const bool any = !aligned16(logits_dev) || ((long long)groups * beams > 1 && (row_stride ? row_stride : vocab) * (dtype == IM_DTYPE_F32 ? 4 : 2) % 16 != 0);
    p.slices = clustered ? clustered : select_slices(dev, groups, beams, vocab);
    p.slice = ((vocab + p.slices - 1) / p.slices + 7) / 8 * 8;
    const long long rows = (long long)groups * beams;
    const size_t need = clustered ? 0 : select_bytes(rows, p.slices, picks);
    IM_REQUIRE(need == 0 || (scratch_dev && aligned16(scratch_dev) && scratch_bytes >= need), "beam selection needs %zu bytes of 16-byte aligned scratch (got %zu)", need,
               scratch_dev ? scratch_bytes : (size_t)0);
    p.x = logits_dev; p.stride = row_stride ? row_stride : vocab;
    p.groups = groups; p.beams = beams; p.vocab = vocab; p.picks = picks;
    p.score = score_dev; p.done = done_dev; p.end_token = end_token;
    p.score_out = score_out_dev; p.parent_out = parent_out_dev; p.token_out = token_out_dev;
    p.part_ms = static_cast<float2 *>(scratch_dev);
    p.part_v = reinterpret_cast<float *>(p.part_ms + rows * p.slices);
    p.part_i = reinterpret_cast<int *>(p.part_v + rows * p.slices * picks);
#define IM_KERNEL(K) \
    (dtype == IM_DTYPE_F32   ? (any ? K<IM_DTYPE_F32, true> : K<IM_DTYPE_F32, false>) \
     : dtype == IM_DTYPE_F16 ? (any ? K<IM_DTYPE_F16, true> : K<IM_DTYPE_F16, false>) \
                             : (any ? K<IM_DTYPE_BF16, true> : K<IM_DTYPE_BF16, false>))
    if (clustered) {
        void (*one)(Select) = IM_KERNEL(beam_cluster_kernel);
        IM_CUDA_CHECK(launch_cluster(one, dim3((unsigned)(rows * p.slices)), dim3(kSelThreads), beams * p.slices, 0, as_stream(stream), p));
        return IM_OK;
    }
    void (*kern)(Select) = IM_KERNEL(beam_slice_kernel);
#undef IM_KERNEL
    IM_CUDA_CHECK(launch_k(kern, dim3(p.slices, (unsigned)rows), dim3(kSelThreads), 0, as_stream(stream), p));
    IM_CUDA_CHECK(launch_k(beam_join_kernel, dim3(groups), dim3(kSelThreads), 0, as_stream(stream), p));
    return IM_OK;
    IM_GUARD_END
}
