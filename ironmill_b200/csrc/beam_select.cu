// The best continuations of a group of beams: value[b, v] = score[b] + x[b, v] - lse[b], lse[b] = log sum_v exp(x[b, v]), the `picks` largest over
// beams and vocabulary, ties to the lowest b * V + v.
//
// The logits are read once, from HBM; what bounds the pass is that read. Within a beam the order of the values is the order of its
// logits, so nothing needs lse before the end: a block walks a slice of a row once for both the running maximum and sum of
// exponentials and the slice's best `picks` logits, and a block per group joins the slices.
//   best of a slice   a thread keeps only the maximum of the elements it meets. The picks-th largest of the threads' maxima, T, is a bound: at
//                     least `picks` elements are >= T. Threads whose maximum reaches T look at their elements again (a few threads, from L2) and
//                     collect those >= T; the rank of each collected element is the number of those before it. Where ties make the collection overflow
//                     the elements are picked one after the other instead.
//   joining           the same with the slices' picks as elements and 64-bit values.
// Sums are f32 per thread over its elements with one running maximum, joined in a fixed order: a run repeats bit by bit, and equal rows
// get equal sums.
#include <cuda_bf16.h>
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "paged.cuh"

namespace im {
namespace {

constexpr int kSelThreads = 256, kSelMost = 64, kSelBuf = 1024;
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

// Rank of a key among n keys in shared memory, larger first; keys differ.
__device__ __forceinline__ bool before(double a, long long ia, double b, long long ib) { return a > b || (a == b && ia < ib); }

// The best of the block: value and index by all threads. `red` holds a value and an index per warp.
__device__ __forceinline__ void block_best(double &v, long long &i, double *red_v, long long *red_i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double v2 = __shfl_xor_sync(0xffffffffu, v, o);
        const long long i2 = __shfl_xor_sync(0xffffffffu, i, o);
        if (before(v2, i2, v, i)) v = v2, i = i2;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red_v[threadIdx.x >> 5] = v, red_i[threadIdx.x >> 5] = i;
    __syncthreads();
    v = red_v[0], i = red_i[0];
    for (int w = 1; w < kSelThreads / 32; w++)
        if (before(red_v[w], red_i[w], v, i)) v = red_v[w], i = red_i[w];
}

// The `picks` best of the elements that visit(f) hands to f(value, index) thread by thread, the same ones at every call, into out_v / out_i in order
// (the rest -inf, -1). top: the largest value this thread hands out. Elements of -inf (and NaN) are none.
template <typename Visit>
__device__ __forceinline__ void pick_best(Visit visit, double top, int picks, double *out_v, long long *out_i) {
    __shared__ double tops[kSelThreads], buf_v[kSelBuf];
    __shared__ long long buf_i[kSelBuf];
    __shared__ double bound;
    __shared__ int count;
    const int t = threadIdx.x;
    tops[t] = top;
    if (t == 0) count = 0, bound = -INFINITY;
    for (int i = t; i < picks; i += kSelThreads) out_v[i] = -INFINITY, out_i[i] = -1;
    __syncthreads();
    int rank = 0;
    for (int j = 0; j < kSelThreads; j++) rank += before(tops[j], j, top, t);
    if (rank == picks - 1) bound = top;
    __syncthreads();
    if (top >= bound && top > -INFINITY)
        visit([&](float v, double value, long long index) {
            if (value >= bound && value > -INFINITY) {
                const int at = atomicAdd(&count, 1);
                if (at < kSelBuf) buf_v[at] = value, buf_i[at] = index;
            }
            (void)v;
        });
    __syncthreads();
    const int n = count;
    if (n <= kSelBuf) {
        for (int i = t; i < n; i += kSelThreads) {
            const double v = buf_v[i];
            const long long x = buf_i[i];
            int r = 0;
            for (int j = 0; j < n && r < picks; j++) r += before(buf_v[j], buf_i[j], v, x);
            if (r < picks) out_v[r] = v, out_i[r] = x;
        }
    } else {
        double last_v = INFINITY;
        long long last_i = -1;
        for (int k = 0; k < picks; k++) {
            double v = -INFINITY;
            long long x = LLONG_MAX;
            visit([&](float, double value, long long index) {
                if (value > -INFINITY && before(last_v, last_i, value, index) && before(value, index, v, x)) v = value, x = index;
            });
            block_best(v, x, buf_v, buf_i);
            if (!(v > -INFINITY)) break;
            if (t == 0) out_v[k] = v, out_i[k] = x;
            last_v = v;
            last_i = x;
        }
    }
    __syncthreads();
}

// grid (slices, rows)
template <int DT>
__global__ void __launch_bounds__(kSelThreads) beam_slice_kernel(const Select p) {
    using L = Logit<DT>;
    using T = typename L::T;
    constexpr int V = L::kVec;
    __shared__ float red_m[kSelThreads / 32], red_s[kSelThreads / 32];
    __shared__ double out_v[kSelMost];
    __shared__ long long out_i[kSelMost];
    pdl_trigger();
    pdl_wait();
    const int slice = blockIdx.x, t = threadIdx.x;
    const long long row = blockIdx.y;
    if (p.done && p.done[row]) return;
    const T *x = static_cast<const T *>(p.x) + row * p.stride;
    const int a = slice * p.slice, b = min(a + p.slice, p.vocab);
    // 16-byte requests from the first aligned element on; what is before and behind them is read one by one
    const int head = min(b - a, (int)((16 - (reinterpret_cast<uintptr_t>(x + a) & 15)) % 16 / sizeof(T)));
    const int vecs = (b - a - head) / V, tail = a + head + vecs * V;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + a + head);
    float m = -INFINITY, s = 0.0f;
    auto take = [&](const float *f, int n) {
        float top = m;
        for (int j = 0; j < n; j++) top = fmaxf(top, f[j]);
        if (top > m) {
            s *= __expf(m - top);
            m = top;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        for (int j = 0; j < n; j++) s += __expf(f[j] - base);
    };
    int i = t;
    for (; i + 3 * kSelThreads < vecs; i += 4 * kSelThreads) {
        uint4 u[4];
#pragma unroll
        for (int k = 0; k < 4; k++) u[k] = ldg_stream_v4(xv + i + k * kSelThreads);
        float f[4 * V];
#pragma unroll
        for (int k = 0; k < 4; k++) L::split(u[k], f + k * V);
        take(f, 4 * V);
    }
    for (; i < vecs; i += kSelThreads) {
        float f[V];
        L::split(ldg_stream_v4(xv + i), f);
        take(f, V);
    }
    for (int e = a + t; e < a + head; e += kSelThreads) {
        const float f = L::get(x[e]);
        take(&f, 1);
    }
    for (int e = tail + t; e < b; e += kSelThreads) {
        const float f = L::get(x[e]);
        take(&f, 1);
    }
    auto visit = [&](auto f) {
        for (int i = t; i < vecs; i += kSelThreads) {
            float g[V];
            L::split(__ldg(xv + i), g);
#pragma unroll
            for (int j = 0; j < V; j++) f(g[j], (double)g[j], (long long)(a + head + i * V + j));
        }
        for (int e = a + t; e < a + head; e += kSelThreads) {
            const float g = L::get(x[e]);
            f(g, (double)g, (long long)e);
        }
        for (int e = tail + t; e < b; e += kSelThreads) {
            const float g = L::get(x[e]);
            f(g, (double)g, (long long)e);
        }
    };
    // joined over lanes, then warps, in a fixed order
    float M = warp_max(m);
    float S = warp_sum(m == -INFINITY && s == 0.0f ? 0.0f : s * __expf(m - M));
    if ((t & 31) == 0) red_m[t >> 5] = M, red_s[t >> 5] = S;
    pick_best(visit, (double)m, p.picks, out_v, out_i);
    if (t == 0) {
        M = -INFINITY;
        for (int w = 0; w < kSelThreads / 32; w++) M = fmaxf(M, red_m[w]);
        S = 0.0f;
        for (int w = 0; w < kSelThreads / 32; w++) S += red_m[w] == -INFINITY && red_s[w] == 0.0f ? 0.0f : red_s[w] * __expf(red_m[w] - M);
        p.part_ms[row * p.slices + slice] = make_float2(M, S);
    }
    const long long at = (row * p.slices + slice) * p.picks;
    for (int k = t; k < p.picks; k += kSelThreads) {
        p.part_v[at + k] = (float)out_v[k];
        p.part_i[at + k] = (int)out_i[k];
    }
}

// grid (groups)
__global__ void __launch_bounds__(kSelThreads) beam_join_kernel(const Select p) {
    __shared__ double offset[kSelMost];  // score - lse of each beam; NaN: nothing of it is picked
    __shared__ double out_v[kSelMost];
    __shared__ long long out_i[kSelMost];
    pdl_trigger();
    pdl_wait();
    const int group = blockIdx.x, t = threadIdx.x, lane = t & 31;
    const long long row0 = (long long)group * p.beams;
    for (int b = t >> 5; b < p.beams; b += kSelThreads / 32) {
        const bool done = p.done && p.done[row0 + b];
        float m = -INFINITY;
        double s = 0.0;
        if (!done) {
            const float2 *ms = p.part_ms + (row0 + b) * p.slices;
            for (int i = lane; i < p.slices; i += 32) m = fmaxf(m, ms[i].x);
            m = warp_max(m);
            for (int i = lane; i < p.slices; i += 32)
                if (!(ms[i].x == -INFINITY && ms[i].y == 0.0f)) s += (double)ms[i].y * exp((double)ms[i].x - (double)m);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        if (lane == 0) {
            const double lse = (double)m + log(s);
            offset[b] = done ? (double)p.score[row0 + b] : lse > -INFINITY && lse < INFINITY ? (double)p.score[row0 + b] - lse : NAN;
        }
    }
    __syncthreads();
    const int per = p.slices * p.picks, n = p.beams * per;
    auto visit = [&](auto f) {
        for (int i = t; i < n; i += kSelThreads) {
            const int b = i / per, k = i - b * per;
            if (p.done && p.done[row0 + b]) {
                if (k == 0) f(0.0f, offset[b], (long long)b * p.vocab + p.end_token);
                continue;
            }
            const float v = p.part_v[row0 * per + i];
            const int token = p.part_i[row0 * per + i];
            if (token >= 0) f(v, offset[b] + (double)v, (long long)b * p.vocab + token);
        }
    };
    double top = -INFINITY;
    visit([&](float, double value, long long) { if (value > top) top = value; });
    pick_best(visit, top, p.picks, out_v, out_i);
    for (int k = t; k < p.picks; k += kSelThreads) {
        const long long i = out_i[k], at = (long long)group * p.picks + k;
        p.score_out[at] = (float)out_v[k];
        p.parent_out[at] = i < 0 ? -1 : (int)(i / p.vocab);
        p.token_out[at] = i < 0 ? -1 : (int)(i % p.vocab);
    }
}

// Slices of a row: about eight blocks of all rows for every SM, none below kSelLeast elements.
int select_slices(const Device *dev, int groups, int beams, int vocab) {
    const long long rows = (long long)groups * beams;
    const long long want = (8ll * dev->sm_count + rows - 1) / rows, most = (vocab + kSelLeast - 1) / kSelLeast;
    return (int)std::max(1ll, std::min(std::min(want, most), 64ll));
}
size_t select_bytes(long long rows, int slices, int picks) { return (size_t)rows * slices * (8 + 8 * (size_t)picks) + 16; }

}  // namespace
}  // namespace im

IM_EXPORT size_t im_cuda_beam_select_scratch_bytes(const im_device *dev, int groups, int beams, int vocab, int picks) {
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
    IM_REQUIRE(reinterpret_cast<uintptr_t>(logits_dev) % (dtype == IM_DTYPE_F32 ? 4 : 2) == 0, "logits are not aligned to their type");
    IM_REQUIRE(!done_dev || (end_token >= 0 && end_token < vocab), "end_token %d of %d", end_token, vocab);
    int rc = paged_device(dev);
    if (rc != IM_OK) return rc;
    if (groups == 0) return IM_OK;
    Select p;
    p.slices = select_slices(dev, groups, beams, vocab);
    p.slice = ((vocab + p.slices - 1) / p.slices + 7) / 8 * 8;
    const long long rows = (long long)groups * beams;
    IM_REQUIRE(scratch_dev && aligned16(scratch_dev) && scratch_bytes >= select_bytes(rows, p.slices, picks), "beam selection needs %zu bytes of 16-byte aligned scratch (got %zu)",
               select_bytes(rows, p.slices, picks), scratch_dev ? scratch_bytes : (size_t)0);
    p.x = logits_dev; p.stride = row_stride ? row_stride : vocab;
    p.groups = groups; p.beams = beams; p.vocab = vocab; p.picks = picks;
    p.score = score_dev; p.done = done_dev; p.end_token = end_token;
    p.score_out = score_out_dev; p.parent_out = parent_out_dev; p.token_out = token_out_dev;
    p.part_ms = static_cast<float2 *>(scratch_dev);
    p.part_v = reinterpret_cast<float *>(p.part_ms + rows * p.slices);
    p.part_i = reinterpret_cast<int *>(p.part_v + rows * p.slices * picks);
    void (*kern)(Select) = dtype == IM_DTYPE_F32 ? beam_slice_kernel<IM_DTYPE_F32> : dtype == IM_DTYPE_F16 ? beam_slice_kernel<IM_DTYPE_F16> : beam_slice_kernel<IM_DTYPE_BF16>;
    IM_CUDA_CHECK(launch_k(kern, dim3(p.slices, (unsigned)rows), dim3(kSelThreads), 0, as_stream(stream), p));
    IM_CUDA_CHECK(launch_k(beam_join_kernel, dim3(groups), dim3(kSelThreads), 0, as_stream(stream), p));
    return IM_OK;
    IM_GUARD_END
}
