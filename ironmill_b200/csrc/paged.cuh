// A paged cache of keys and values as its kernels see it (paged_cache.cu, paged_attn.cu).
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace im {

struct PagedView {
    long long layer_stride, page_stride;  // elements
    int layers, pages, nkv, page, hd, nseq, width;
    long long table_stride;
    int rows;  // most rows of a sequence: width * page
    const int *table, *len;

    // rows of a sequence before the new tokens: a length that the table cannot hold counts as the nearest one that it can
    __device__ __forceinline__ int length(int seq) const { return min(max(__ldg(len + seq), 0), rows); }
    // element offset of slot 0 of head 0 in the page that holds row r, -1 where there is none; r in [0, rows)
    __device__ __forceinline__ long long page_of(int seq, int r) const {
        const int p = __ldg(table + seq * table_stride + r / page);
        return (unsigned)p < (unsigned)pages ? p * page_stride : -1;
    }
    __device__ __forceinline__ long long row_of(int seq, int r) const {  // of head 0; + h * page * hd for head h
        if ((unsigned)r >= (unsigned)rows) return -1;
        const long long at = page_of(seq, r);
        return at < 0 ? -1 : at + (long long)(r % page) * hd;
    }
};

// Whether two arrays share memory; sizes in bytes.
inline bool share_memory(const void *a, long long na, const void *b, long long nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}
// Whether n rows of `row` bytes, sa bytes apart from a on, share memory with such rows sb apart from b on. Rows of the same stride may lie between one
// another; of others it is their whole span that counts.
inline bool share_rows(const void *a, long long sa, const void *b, long long sb, long long row, long long n) {
    const auto span = [&](long long stride) { return (n - 1 > (1ll << 60) / stride ? 1ll << 60 : (n - 1) * stride) + row; };
    if (n < 1 || !share_memory(a, span(sa), b, span(sb))) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    const long long d = (long long)((x < y ? y - x : x - y) % (uintptr_t)sa);
    return sa != sb || d < row || sa - d < row;
}
inline bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Checks what the host can see of a cache and fills the kernels' view; layer < 0: all of them.
int paged_view(const im_paged_kv *kv, int layer, PagedView *out);
// The handle's device has to be the current one: launches and attributes go there.
int paged_device(const im_device *dev);

// The sequence of a token: the last s with start[s] <= token, by a warp, 32 places at a time.
__device__ __forceinline__ int paged_seq_of(const int *start, int nseq, int token) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = nseq;  // it lies in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const unsigned le = __ballot_sync(0xffffffffu, at < lo + n && __ldg(start + at) <= token);
        const int k = max(__popc(le) - 1, 0);
        n = min(step, n - k * step);
        lo += k * step;
        if (n <= 0) return lo;
    }
    return lo;
}

template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t u) {
    if (BF16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <bool BF16>
__device__ __forceinline__ float one16(const uint16_t *p) {
    const uint32_t u = *p;
    return BF16 ? __uint_as_float(u << 16) : __half2float(__ushort_as_half((unsigned short)u));
}

}  // namespace im
