// What the kernels share that read a paged cache into the tcgen05 tensor cores (paged_attn_tc.cu, paged_weights.cu).
#pragma once
#include "paged_attn.cuh"

namespace im {

// warps 0-7: weights or sums; 8: products; 9-12: copies
constexpr int kTcTile = 128, kTcThreads = 13 * 32, kTcMma = 8, kTcCopy = 9, kTcCopyWarps = 4;

// The items of a CTA's share, one after the other; every warp walks them for itself.
template <int R, int MODE>
struct Items {
    const PagedAttn &p;
    const int units;
    int unit, head, tile;
    long long left;
    PagedUnit u;
    int tiles, t0, t1, index;
    __device__ __forceinline__ Items(const PagedAttn &p, int units, const Share &s, const PagedUnit &first)
        : p(p), units(units), unit(s.unit - 1), head(p.kv.nkv - 1), tile(0), left(s.to - s.from), tiles(0), t0(0), t1(0), index(-1) {
        if (left > 0) {
            unit = s.unit;
            head = s.head - 1;
            u = first;
            tiles = unit_tiles<kTcTile, MODE>(u);
            tile = s.tile;
        }
    }
    __device__ __forceinline__ bool next() {
        if (left <= 0) return false;
        if (++head == p.kv.nkv) {
            head = 0;
            do {
                if (++unit >= units) return false;
                u = paged_unit<R, MODE>(p, unit);
                tiles = unit_tiles<kTcTile, MODE>(u);
            } while (tiles == 0);
        }
        t0 = tile;
        t1 = (int)min((long long)tiles, t0 + left);
        left -= t1 - t0;
        tile = 0;
        index++;
        return true;
    }
};

// Products and commits of one lane (`one`) of a converged warp: what they name is the same in all lanes, and uniform() says so where the compiler
// cannot see it; from registers of a single lane it would move every operand of every product to a uniform register first.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ uint32_t elected() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}\n" : "=r"(one));
    return one;
}
__device__ __forceinline__ void umma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(one)
                 : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {  // A operand in tensor memory
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(one)
                 : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t one, uint64_t *bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)), "r"(one)
                 : "memory");
}
// The 256 threads of both sets of four warps.
__device__ __forceinline__ void both_halves() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
// What copies of other threads have written, once their barrier says so, before the tensor cores read it.
__device__ __forceinline__ void copies_landed() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

}  // namespace im
