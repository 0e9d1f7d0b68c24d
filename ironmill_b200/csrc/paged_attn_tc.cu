// Attention over a paged cache on the 5th-generation tensor cores, for many rows (token, query head) of a KV head: trees and portions of prompts.
//
// One CTA per SM walks an equal share of the list of all (row tile, KV head) items' tiles of 128 positions (paged_attn.cu has the scheme; a second launch joins
// what the cuts divide). Two sets of four warps ("halves") turn scores into weights, a row per thread; while one of them works, the other's products run:
//     S = Q K^T    both operands in shared memory, accumulator in tensor memory (f32)
//     P = exp2(S)  to registers, running maximum and sum in f32, weights back over the scores in 16 bits (up to 128 rows: as two terms, the weight and what
//                  its rounding left)
//     O += P V     P from tensor memory, V with the head dimension contiguous
// A tile of up to 256 rows (WIDE): the halves own 128 rows each and every tile of K and V serves both. Up to 128 rows: the halves own the even
// and the odd tiles of the share, with accumulators of their own that are joined where the item ends. There the copies set the pace and the second
// term of the weights is free; in a wide tile the chain of scores, weights and products does, and one term is what it takes: half a step of
// a weight (2^-8 bf16, 2^-11 fp16, relative) moves an output by at most that share of the sum of its weights times |values|, as much as rounding the output
// does where all values have one sign, more where they cancel.
// A row's accumulator is rescaled only when its maximum has grown by more than a power of two (as in flash_tc.cu), 2^8 for bf16, 2^3 for fp16.
//
// K, V and queries come by 16-byte cp.async of four warps, rows looked up in the page table: any page size, rows that are not there are zeros and
// known to be none (a bit per row). The copies run ahead over the ends of items as far as the slots allow.
//
// Bounds. Up to 128 rows: the copies, 3200 clocks a tile of 64 KB (20 bytes a clock and SM, 5.6 TB/s). Eight sequences of up to 4001 rows, 34 us: 5.6 until a
// CTA's first scores, 12.6 its tiles, 3.6 its outputs, 5.1 until the slowest CTA is there, 1.3 until the join starts, 5.6 the join. WIDE: a half's chain, 2600
// clocks of weights and as many for its products (64 clocks each), while the other half has its turn: a sequence of 100003 rows and 256 rows of queries 141 us,
// 2.9 TB/s, 745 TFLOP/s. The loops are short on purpose: unrolled, the three kinds of warps waited for instructions more than for anything else (286 us
// against 200 then).
//
// All waits are bounded: one that runs out sets the device error word, every warp then runs to its end.
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "paged_attn.cuh"

namespace im {
namespace {

// warps 0-7: weights; 8: products; 9-12: copies
constexpr int kTcTile = 128, kTcThreads = 13 * 32, kTcMma = 8, kTcCopy = 9, kTcCopyWarps = 4;
// Growth of a row's maximum (in powers of two) that is left in the weights; power of two that a weight has at the maximum: fp16 weights come up to 2^15, so that
// they are normal numbers down to 2^-26 of the maximum (exact to 2^-37 below). bf16 has the range of f32. (A growth
// of 2^8 left in fp16 too: 120.3 us instead of 125.8 for 256 rows over 100003 positions where the scores' spread is four nats, no difference at one.)
constexpr float tc_lazy(bool bf16) { return bf16 ? 8.0f : 3.0f; }
constexpr float tc_lift(bool bf16) { return bf16 ? 0.0f : 12.0f; }

template <int KB, bool WIDE>
struct TcShape {
    static constexpr int kRows = WIDE ? 256 : 128;
    static constexpr int kBlock = 128 * 128;  // bytes of 128 rows of 64 columns
    static constexpr int kQ = (WIDE ? 2 : 1) * KB * kBlock, kSlot = KB * kBlock;
    static constexpr int kK = 3, kV = WIDE ? 2 : 3;  // slots
    static constexpr int kBars = 2 * kK + 2 * kV + 2 + 2 + 4 + 2 + 2;
    static constexpr int kSmall = 8 * 16 + 128 * 8 + kTcCopyWarps * 32 * 8 + kBars * 8 + 48;  // presence bits, maxima and sums, offsets, barriers, address
    static constexpr int kTiles = kQ + (kK + kV) * kSlot;
    static constexpr int kSmem = (kSmall + 1023) / 1024 * 1024 + kTiles;
    static_assert(kSmem <= 232448, "shared memory of an SM");
};

// The items of a CTA's share, one after the other; every warp walks them for itself.
template <int R>
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
            tiles = unit_tiles<kTcTile>(u);
            tile = s.tile;
        }
    }
    __device__ __forceinline__ bool next() {
        if (left <= 0) return false;
        if (++head == p.kv.nkv) {
            head = 0;
            do {
                if (++unit >= units) return false;
                u = paged_unit<R>(p, unit);
                tiles = unit_tiles<kTcTile>(u);
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

// Bit j: the t-th new token sees position pos + j (32 of them); the rows' being there is another matter.
__device__ __forceinline__ uint32_t sees32(const PagedAttn &p, const PagedUnit &u, int t, int pos) {
    const int d = pos - u.len;
    if (d + 32 <= 0) return 0xffffffffu;
    if (d >= u.fresh) return 0u;
    const int from = max(d, 0), shift = from - d;  // bits below `shift` are rows before the new ones
    uint32_t bits;
    if (!p.mask) {
        const int n = t + 1 - from;
        bits = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1;
    } else {
        const uint64_t *m = p.mask + (long long)(u.tok0 + t) * p.mask_words;
        const int w = from >> 6, s = from & 63;
        uint64_t x = w < p.mask_words ? __ldg(m + w) >> s : 0;
        if (s > 32 && w + 1 < p.mask_words) x |= __ldg(m + w + 1) << (64 - s);
        bits = (uint32_t)x;
    }
    const int n = u.fresh - from;
    if (n < 32) bits &= (1u << n) - 1;
    return shift == 0 ? bits : bits << shift | ((1u << shift) - 1);
}

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
// Two f32 side by side.
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 of_two(uint64_t x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// The 256 threads of both halves.
__device__ __forceinline__ void both_halves() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
// What copies of other threads have written, once their barrier says so, before the tensor cores read it.
__device__ __forceinline__ void copies_landed() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Sums of weighted values that a share leaves: four columns of all rows after another, since a warp that writes (and one that joins) has a row per lane.
template <int R>
__device__ __forceinline__ float *tc_part(float *part_o, size_t slot, int hd, int row, int col) { return part_o + (slot * (hd / 4) + col / 4) * (R * 4) + row * 4 + col % 4; }

template <bool BF16, int KB, bool WIDE>
__global__ void __launch_bounds__(kTcThreads, 1) paged_tc_kernel(const __grid_constant__ PagedAttn p, int units, int *err) {
    using Shape = TcShape<KB, WIDE>;
    constexpr int kTerms = WIDE ? 1 : 2;  // 16-bit terms of a weight
    constexpr float kLazy = tc_lazy(BF16), kLift = tc_lift(BF16);
    constexpr int R = Shape::kRows, HD = 64 * KB, SK = Shape::kK, SV = Shape::kV, BLK = Shape::kBlock;
    extern __shared__ __align__(16) unsigned char tc_smem[];
    uint32_t *there = reinterpret_cast<uint32_t *>(tc_smem);                   // [8 tiles][4]: bit j of word w: row 32 w + j of the tile is in the cache
    float2 *ml = reinterpret_cast<float2 *>(there + 32);                       // [128]: maxima and sums, from half to half (not WIDE)
    long long *offs = reinterpret_cast<long long *>(ml + 128);                 // [copying warps][32]: where the rows that a warp copies lie
    uint64_t *kfull = reinterpret_cast<uint64_t *>(offs + kTcCopyWarps * 32), *kempty = kfull + SK, *vfull = kempty + SK, *vempty = vfull + SV, *qfull = vempty + SV,
             *qempty = qfull + 1, *sfull = qempty + 1, *pfull = sfull + 2, *ofull = pfull + 4, *oempty = ofull + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(oempty + 2);
    uint32_t *odd_rows = tmem_slot + 1;  // [4 warps]
    // (shared memory starts at a multiple of 1024: checked, the tiles would not fit otherwise)
    unsigned char *Qs = tc_smem + (Shape::kSmem - Shape::kTiles), *Ks = Qs + Shape::kQ, *Vs = Ks + SK * Shape::kSlot;
    if (smem_u32(Qs) % 1024 != 0) {
        if (threadIdx.x == 0) atomicExch(err, 1);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < SK; i++) {
            mbar_init(&kfull[i], kTcCopyWarps * 33);  // threads whose copies are there; warps that have said which rows are
            mbar_init(&kempty[i], 1);
        }
        for (int i = 0; i < SV; i++) {
            mbar_init(&vfull[i], kTcCopyWarps * 32);
            mbar_init(&vempty[i], 1);
        }
        mbar_init(qfull, kTcCopyWarps * 32);
        mbar_init(qempty, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sfull[i], 1);
            mbar_init(&pfull[2 * i], 4);
            mbar_init(&pfull[2 * i + 1], 4);
            mbar_init(&ofull[i], 1);
            mbar_init(&oempty[i], 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kTcMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = uniform(*tmem_slot);
    pdl_trigger();  // after the allocation: a successor on this SM cannot take the columns first
    pdl_wait();
    PagedUnit at;
    const Share share = units <= 32 ? warp_share<R, kTcTile>(p, units, at) : find_share<R, kTcTile, kTcThreads>(p, units, reinterpret_cast<long long *>(Qs), at);  // (the copies start behind its last barrier)
    Items<R> it(p, units, share, at);
    bool ok = true;
    if (warp >= kTcCopy) {
        // ---- copies: this warp's 32 rows of every 128
        const int w0 = (warp - kTcCopy) * 32;
        long long *mine = offs + w0;
        auto room = [&](uint64_t *bar, uint32_t parity) {
            if (ok && !mbar_try_wait(bar, parity)) ok = wait_for(bar, parity, err);
            __syncwarp();
        };
        auto requested = [&](uint64_t *bar) {  // each thread arrives when what it has requested is there
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
        };
        // 32 rows whose offsets (elements from base; -1: none) are in mine[]
        auto rows32 = [&](unsigned char *dst, const uint16_t *base) {
            constexpr int CH = 8 * KB, RPI = 32 / CH;
            const int c = lane % CH, r0 = lane / CH;
            const uint32_t at = smem_u32(dst) + (c >> 3) * BLK + (w0 + r0) * 128;
#pragma unroll 1
            for (int i0 = 0; i0 < 32 / RPI; i0 += 8) {
                long long o[8];
#pragma unroll
                for (int i = 0; i < 8; i++) o[i] = mine[(i0 + i) * RPI + r0];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int r = (i0 + i) * RPI;
                    cp16(at + r * 128 + (((c & 7) ^ ((r + r0) & 7)) << 4), base + (o[i] < 0 ? 0 : o[i] + c * 8), o[i] >= 0);
                }
            }
        };
        auto place = [&](long long o) {
            __syncwarp();
            mine[lane] = o;
            __syncwarp();
        };
        int kc = 0, vc = 0;
        auto lookup = [&](const PagedUnit &u, int head, int pos) -> long long {
            if (pos >= u.end) return -1;
            const long long o = p.kv.row_of(u.seq, pos);
            return o < 0 ? -1 : o + (long long)head * p.kv.page * HD;
        };
        while (it.next()) {
            const PagedUnit &u = it.u;
            long long o = lookup(u, it.head, it.t0 * kTcTile + w0 + lane);
            if (it.index > 0) room(qempty, (it.index - 1) & 1);
            for (int h = 0; h < (WIDE && u.rows > 128 ? 2 : 1); h++) {
                const int r = h * 128 + w0 + lane;
                place(r < u.rows ? (u.tok0 + (u.row0 + r) / p.group) * p.qs + (long long)(it.head * p.group + (u.row0 + r) % p.group) * HD : -1);
                rows32(Qs + h * KB * BLK, p.q);
            }
            requested(qfull);
            for (int t = it.t0; t < it.t1; t++) {
                const int ks = kc % SK, vs = vc % SV;
                // the places of the next tile's rows are looked up while this one is requested
                const long long next = t + 1 < it.t1 ? lookup(u, it.head, (t + 1) * kTcTile + w0 + lane) : -1;
                if (kc >= SK) room(&kempty[ks], (kc / SK - 1) & 1);
                const unsigned word = __ballot_sync(0xffffffffu, o >= 0);
                if (lane == 0) {
                    there[(kc & 7) * 4 + w0 / 32] = word;
                    mbar_arrive(&kfull[ks]);
                }
                place(o);
                rows32(Ks + ks * Shape::kSlot, p.kc);
                requested(&kfull[ks]);
                kc++;
                if (vc >= SV) room(&vempty[vs], (vc / SV - 1) & 1);
                rows32(Vs + vs * Shape::kSlot, p.vc);
                requested(&vfull[vs]);
                vc++;
                o = next;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == kTcMma) {
        // ---- products: one thread waits and issues them all; what it does between them is kept short, the tensor cores' queue holds only a few.
        // Instruction descriptors as in flash_tc.cu: f32 accumulator, fp16 (0) or bf16 (1) operands in bits 7-9 and 10-12, B MN-major in bit 16, N >> 3 in
        // bits 17-22, M >> 4 in bits 24-28
        constexpr uint32_t kType = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(128 >> 4) << 24);
        constexpr uint32_t kS = kType | ((uint32_t)(kTcTile >> 3) << 17), kPV = kType | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
        {
            const uint32_t one = elected();
            const uint64_t qd = desc_sw128(smem_u32(Qs), 16), kd = desc_sw128(smem_u32(Ks), 16), vd = desc_sw128(smem_u32(Vs), BLK);
            int ks = 0, vs = 0, turn0 = 0, turn1 = 0;     // slots; weights of the halves that were waited for
            int used0 = 0, used1 = 0;                     // items that the halves' accumulators were used for
            uint32_t kturn = 0, vturn = 0;                // parities of the slots' turns
            auto wait = [&](uint64_t *bar, uint32_t parity) {
                if (ok && !mbar_try_wait(bar, parity)) ok = wait_for(bar, parity, err);
                __syncwarp();
            };
            auto scores = [&](int h) {
                copies_landed();
                fence_after();
                if (!ok) return;
                const uint64_t a = qd + (WIDE && h ? KB * BLK / 16 : 0), b = kd + ks * (Shape::kSlot / 16);
#pragma unroll
                for (int j = 0; j < KB * 4; j++) umma_ss(one, tmem + (uint32_t)(h * kTcTile), a + (j / 4 * BLK + (j & 3) * 32) / 16, b + (j / 4 * BLK + (j & 3) * 32) / 16, kS, j > 0);
                umma_commit(one, &sfull[h]);
            };
            auto values = [&](int h, bool first, bool last) {
                const uint32_t w = tmem + (uint32_t)(h * kTcTile), o = tmem + 256u + (uint32_t)(h * 128), turn = (h ? turn1 : turn0) & 1;
                const uint64_t b = vd + vs * (Shape::kSlot / 16);
#pragma unroll 1
                for (int c = 0; c < 2; c++) {  // 64 positions: 32 columns of the weights' first terms, 32 of the second
                    wait(&pfull[2 * h + c], turn);
                    copies_landed();
                    fence_after();
                    if (!ok) return;
#pragma unroll
                    for (int i = 0; i < 4 * kTerms; i++)
                        umma_ts(one, o, w + (uint32_t)(c * 64 + i % kTerms * 32 + i / kTerms * 8), b + (c * 4 + i / kTerms) * (2048 / 16), kPV, i > 0 || c > 0 || !first);
                }
                turn0 += !h;
                turn1 += h;
                if (last) umma_commit(one, &ofull[h]);
            };
            auto release = [&](uint64_t *bar) {  // once the products issued so far are done
                if (ok) umma_commit(one, bar);
            };
            auto k_done = [&]() {
                release(&kempty[ks]);
                if (++ks == SK) ks = 0, kturn ^= 1;
            };
            auto v_done = [&]() {
                release(&vempty[vs]);
                if (++vs == SV) vs = 0, vturn ^= 1;
            };
            while (it.next()) {
                const int T = (int)uniform(it.t1 - it.t0);
                wait(qfull, it.index & 1);
                auto drained = [&](int halves) {  // the outputs of the item before that these halves had rows of have been read
                    if (used0 > 0) wait(&oempty[0], (used0 - 1) & 1);
                    used0++;
                    if (halves < 2) return;
                    if (used1 > 0) wait(&oempty[1], (used1 - 1) & 1);
                    used1++;
                };
                if constexpr (WIDE) {
                    const int halves = (int)uniform(it.u.rows > 128 ? 2 : 1);
#pragma unroll 1
                    for (int t = 0; t <= T; t++) {
                        if (t == 1) drained(halves);
#pragma unroll 1
                        for (int h = 0; h < halves; h++) {
                            if (t > 0) {
                                if (h == 0) wait(&vfull[vs], vturn);
                                values(h, t == 1, t == T);
                            }
                            if (t < T) {
                                if (h == 0) wait(&kfull[ks], kturn);
                                scores(h);
                            }
                        }
                        if (t > 0) v_done();
                        if (t < T) k_done();
                        if (t == T - 1) release(qempty);
                    }
                } else {
#pragma unroll 1
                    for (int t = 0; t < T + 2; t++) {
                        if (t == 2) drained(2);
                        if (t >= 2) {
                            wait(&vfull[vs], vturn);
                            values(t & 1, t < 4, t >= T);
                            v_done();
                        }
                        if (t < T) {
                            wait(&kfull[ks], kturn);
                            scores(t & 1);
                            k_done();
                        }
                        if (t == T - 1) release(qempty);
                    }
                }
            }
        }
        __syncwarp();
    } else {
        // ---- weights: a row per thread
        const int h = warp >> 2, r = (warp & 3) * 32 + lane, R_ = WIDE ? h * 128 + r : r;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + (uint32_t)(h * kTcTile), to = tmem + lanes + 256u + (uint32_t)(h * 128);
        const float scale = fabsf(p.scale2);
        int seen = 0, tiles_before = 0, finished = 0;  // scores of this half; tiles and items with tiles of the half so far
        while (it.next()) {
            const PagedUnit &u = it.u;
            const int T = it.t1 - it.t0, jobs = WIDE ? (u.rows > h * 128 ? T : 0) : (T - h + 1) / 2;
            const int token = (u.row0 + min(R_, u.rows - 1)) / p.group;
            float m = -INFINITY, l = 0.0f;
            for (int job = 0; job < jobs; job++) {
                const int t = WIDE ? job : 2 * job + h;
                if (ok && !wait_for(&sfull[h], seen & 1, err)) ok = false;
                seen++;
                fence_after();
                const int p0 = (it.t0 + t) * kTcTile;
                const uint32_t *rows = there + ((tiles_before + t) & 7) * 4;
                const bool part = (rows[0] & rows[1] & rows[2] & rows[3]) != 0xffffffffu || p0 + kTcTile > u.len;  // some row does not see all of the tile
                float top = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < kTcTile; c += 64) {
                    float s[64];
                    ld32(ts + (uint32_t)c, reinterpret_cast<uint32_t *>(s));
                    ld32(ts + (uint32_t)c + 32u, reinterpret_cast<uint32_t *>(s) + 32);
                    tmem_wait_ld();
                    if (part || p.scale2 < 0.0f) {
                        const float sign = p.scale2 < 0.0f ? -1.0f : 1.0f;
                        const uint32_t w0 = rows[c / 32] & sees32(p, u, token, p0 + c), w1 = rows[c / 32 + 1] & sees32(p, u, token, p0 + c + 32);
#pragma unroll
                        for (int j = 0; j < 64; j++) s[j] = (j < 32 ? w0 : w1) >> (j & 31) & 1u ? s[j] * sign : -INFINITY;
                        st32(ts + (uint32_t)c, reinterpret_cast<uint32_t *>(s));
                        st32(ts + (uint32_t)c + 32u, reinterpret_cast<uint32_t *>(s) + 32);
                    }
                    float mx[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) mx[j] = s[j];
#pragma unroll
                    for (int j = 4; j < 64; j++) mx[j & 3] = fmaxf(mx[j & 3], s[j]);
                    top = fmaxf(fmaxf(top, fmaxf(mx[0], mx[1])), fmaxf(mx[2], mx[3]));
                }
                top *= scale;
                if (__any_sync(0xffffffffu, top > m + kLazy)) {  // (-inf + anything is -inf: a row's first visible position is one)
                    const float m_new = fmaxf(m, top), corr = m_new == -INFINITY ? 1.0f : ex2(m - m_new);
                    m = m_new;
                    l *= corr;
                    if (job > 0) {
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            ld32(to + (uint32_t)c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
                            st32(to + (uint32_t)c, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.0f : m - kLift;
                tmem_wait_st();
                const uint64_t scale_two = two(scale, scale), base_two = two(-base, -base), minus_one = two(-1.0f, -1.0f);
                uint64_t sum[2] = {0, 0};
#pragma unroll 1
                for (int c = 0; c < kTcTile; c += 64) {  // weights of 64 positions over their scores: first terms, second terms
                    uint32_t s[64];
                    ld32(ts + (uint32_t)c, s);
                    ld32(ts + (uint32_t)c + 32u, s + 32);
                    tmem_wait_ld();
#pragma unroll
                    for (int h2 = 0; h2 < 2; h2++) {
                        uint32_t w[16], w2[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const float2 e = of_two(fma_two(two(__uint_as_float(s[32 * h2 + 2 * j]), __uint_as_float(s[32 * h2 + 2 * j + 1])), scale_two, base_two));
                            const float x0 = ex2(e.x), x1 = ex2(e.y);
                            const uint64_t x = two(x0, x1);
                            sum[j & 1] = add_two(sum[j & 1], x);
                            w[j] = pack2<BF16>(x0, x1);
                            if (kTerms == 1) continue;
                            const float2 back = unpack2<BF16>(w[j]);
                            const float2 left = of_two(fma_two(two(back.x, back.y), minus_one, x));
                            w2[j] = pack2<BF16>(left.x, left.y);
                        }
                        st16(ts + (uint32_t)(c + 16 * h2), w);
                        if (kTerms > 1) st16(ts + (uint32_t)(c + 32 + 16 * h2), w2);
                    }
                    tmem_wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&pfull[2 * h + c / 64]);
                }
                const float2 sums = of_two(add_two(sum[0], sum[1]));
                l += sums.x + sums.y;
            }
            tiles_before += T;
            // ---- the item's (or the share's part of it) rows
            if (jobs > 0 && ok && !wait_for(&ofull[h], finished & 1, err)) ok = false;
            finished += jobs > 0;
            float f0 = 1.0f, f1 = 0.0f;
            if constexpr (!WIDE) {  // each half takes half of the columns, of both accumulators
                const float2 mine = make_float2(m, l);
                float2 o;
                fence_before();
                if (h) {  // (one place for a row, where each half finds what the other one has)
                    ml[r] = mine;
                    both_halves();
                    both_halves();
                    o = ml[r];
                } else {
                    both_halves();
                    o = ml[r];
                    ml[r] = mine;
                    both_halves();
                }
                const float M = fmaxf(m, o.x);
                f0 = m == -INFINITY && l == 0.0f ? 0.0f : ex2(m - M);
                f1 = o.x == -INFINITY && o.y == 0.0f ? 0.0f : ex2(o.x - M);
                // (added in the order of the halves, by both of them)
                const float own = f0 == 0.0f ? 0.0f : l * f0, other = f1 == 0.0f ? 0.0f : o.y * f1;
                l = h ? other + own : own + other;
                m = M;
            }
            fence_after();
            const bool live = R_ < u.rows && ok;
            const bool whole = it.t0 == 0 && it.t1 == it.tiles;
            const size_t slot = (size_t)blockIdx.x * 2 + (it.index == 0 ? 0 : 1);
            if (tid == 0) note_span(p, it.unit, it.head, it.t0, it.t1, it.tiles, blockIdx.x, it.index == 0 ? 0 : 1);
            const float inv = whole ? (l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l) : 1.0f;
            uint16_t *out = p.out + (u.tok0 + token) * p.os + (long long)(it.head * p.group + (u.row0 + min(R_, u.rows - 1)) % p.group) * HD;
            float worst = 0.0f;
            bool any_other = false;  // (a half without tiles has left nothing)
            const uint32_t other_half = tmem + lanes + 256u + (uint32_t)((1 - h) * 128);
            if (WIDE ? jobs > 0 : true) {
#pragma unroll 1
                for (int c = WIDE ? 0 : h * (HD / 2); c < (WIDE ? HD : (h + 1) * (HD / 2)); c += 32) {
                    uint32_t a[32];
                    float v[32];
                    ld32(to + (uint32_t)c, a);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; j++) v[j] = f0 == 0.0f ? 0.0f : __uint_as_float(a[j]) * f0;
                    if (!WIDE && f1 != 0.0f) any_other = true;
                    if (!WIDE && __any_sync(0xffffffffu, any_other)) {
                        ld32(other_half + (uint32_t)c, a);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; j++) v[j] += f1 == 0.0f ? 0.0f : __uint_as_float(a[j]) * f1;
                    }
#pragma unroll
                    for (int j = 0; j < 32; j++) worst += v[j] * 0.0f;  // zero unless a value is not finite
                    if (!live) continue;
                    if (whole) {
#pragma unroll
                        for (int j = 0; j < 32; j += 8)
                            *reinterpret_cast<uint4 *>(out + c + j) = make_uint4(pack2<BF16>(v[j] * inv, v[j + 1] * inv), pack2<BF16>(v[j + 2] * inv, v[j + 3] * inv),
                                                                                 pack2<BF16>(v[j + 4] * inv, v[j + 5] * inv), pack2<BF16>(v[j + 6] * inv, v[j + 7] * inv));
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(tc_part<R>(p.part_o, slot, HD, R_, c + j)) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                    }
                }
            }
            fence_before();
            __syncwarp();
            // (a wide tile's half without rows has nothing to wait for, and must not run ahead of the products' waits by phases of its own)
            if (lane == 0 && (!WIDE || jobs > 0)) mbar_arrive(&oempty[h]);
            // Rows whose sums are not finite are noted and left to the joining launch: nothing here waits for them
            unsigned bad = __ballot_sync(0xffffffffu, live && !(worst == 0.0f));
            if constexpr (!WIDE) {  // the first half's warps note what either found
                if (h && lane == 0) odd_rows[warp & 3] = bad;
                both_halves();
                if (!h) bad |= odd_rows[warp];
            }
            if (WIDE || h == 0) {
                if (whole && lane == 0) p.odd[((long long)it.unit * p.kv.nkv + it.head) * 8 + warp] = bad;
                if (live && !whole) p.part_ml[slot * R + R_] = make_float2(m - kLift, bad >> lane & 1u ? NAN : l);
            }
        }
    }
    fence_before();
    sync_and_settle(ok);
    if (warp == kTcMma) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

constexpr int kTcJoinThreads = 128, kTcJoinWarps = kTcJoinThreads / 32;
// Rows 32 * rows + j of an item, j a bit of `bad`, from the positions they see alone: every `warps`-th of them, by a warp. (By itself and from numbers
// alone: what it needs of registers and memory is no cost where no row is odd.)
template <bool BF16, int R, int HD>
__device__ __noinline__ void odd_rows_again(const PagedAttn &p, int unit, int head, int rows, unsigned bad, int warp, int warps) {
    const int lane = threadIdx.x & 31;
    const PagedUnit u = paged_unit<R>(p, unit);
#pragma unroll 1
    for (int n = 0; bad; n++, bad &= bad - 1) {
        if (n % warps != warp) continue;
        const int r = rows * 32 + __ffs(bad) - 1;
        float o[HD / 32], m, l;
        plain_row<BF16, HD>(p, u, head, r, 0, u.end, o, m, l);
        const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
        uint16_t *out = p.out + (u.tok0 + (u.row0 + r) / p.group) * p.os + (long long)(head * p.group + (u.row0 + r) % p.group) * HD + lane;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) out[32 * i] = (uint16_t)pack2<BF16>(o[i] * inv, 0.0f);
    }
}

// Four columns of row r of an item that a cut divides. Returns the lanes whose rows are not finite: those are not written.
template <bool BF16, int HD, int R, int N>
__device__ __forceinline__ unsigned join_parts(const PagedAttn &p, const PagedUnit &u, int2 span, int head, int r, int c) {
    const bool live = r < u.rows;
    const int first = span.x >> 1, parts = span.y - first + 1, at = min(r, u.rows - 1);
    float M = -INFINITY, L = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int i0 = 0; i0 < parts; i0 += N) {
        float2 x[N];
        float4 v[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int k = min(i0 + i, parts - 1);
            const size_t slot = k == 0 ? (size_t)span.x : (size_t)(first + k) * 2;
            x[i] = p.part_ml[slot * R + at];
            v[i] = *reinterpret_cast<const float4 *>(tc_part<R>(p.part_o, slot, HD, at, c));
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (i0 + i >= parts) x[i] = make_float2(-INFINITY, 0.0f);
            top = fmaxf(top, x[i].x);
        }
        const float corr = M == top ? 1.0f : ex2(M - top);
        M = top;
        L *= corr;
        o = make_float4(o.x * corr, o.y * corr, o.z * corr, o.w * corr);
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (x[i].x == -INFINITY && x[i].y == 0.0f) continue;  // nothing seen in this part
            const float f = ex2(x[i].x - top);
            L += x[i].y * f;
            o.x += v[i].x * f; o.y += v[i].y * f; o.z += v[i].z * f; o.w += v[i].w * f;
        }
    }
    const unsigned bad = __ballot_sync(0xffffffffu, live && L != L);
    if (!live || L != L) return bad;
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    const int t = (u.row0 + r) / p.group, g = (u.row0 + r) % p.group;
    *reinterpret_cast<uint2 *>(p.out + (u.tok0 + t) * p.os + (long long)(head * p.group + g) * HD + c) = make_uint2(pack2<BF16>(o.x * inv, o.y * inv), pack2<BF16>(o.z * inv, o.w * inv));
    return bad;
}

// Items that a cut divides: a warp per 32 rows and four columns, a row per lane. Blocks are small enough to wait beside a CTA of the kernel above.
// Rows that it has noted as not finite, of any item, are done again: the warps of 32 rows share them. (In the kernel above, where a warp had them one
// after the other at 1.4 us a position, other warps ran out of patience. 32 rows of each of 128 items over 1000 positions: 45 ms there, 0.9 here.)
// No shared memory and few registers: the kernel above leaves little of them free (with 2 KB a block eight portions of 128 tokens behind 500 took 44.9 us, 43.4 so).
template <bool BF16, int KB, bool WIDE>
__global__ void __launch_bounds__(kTcJoinThreads, WIDE ? 9 : 12) paged_tc_join_kernel(const __grid_constant__ PagedAttn p) {
    constexpr int R = TcShape<KB, WIDE>::kRows, HD = 64 * KB, N = WIDE ? 8 : 4;  // N: parts that are requested together
    pdl_trigger();
    pdl_wait();
    const int item = blockIdx.x, unit = item / p.kv.nkv, head = item - unit * p.kv.nkv, lane = threadIdx.x & 31;
    const int w = blockIdx.y * kTcJoinWarps + (threadIdx.x >> 5), rows = w / (HD / 4), r = rows * 32 + lane, c = w % (HD / 4) * 4;
    const int2 span = *reinterpret_cast<const int2 *>(p.spans + 2 * (long long)item);
    const PagedUnit u = paged_unit<R>(p, unit);
    if (rows * 32 >= u.rows) return;  // (a unit without tiles has no rows)
    const unsigned bad = span.x < 0 ? p.odd[(long long)item * 8 + rows] : join_parts<BF16, HD, R, N>(p, u, span, head, r, c);
    if (bad) odd_rows_again<BF16, R, HD>(p, unit, head, rows, bad, w % (HD / 4), HD / 4);
}

template <bool BF16, int KB, bool WIDE>
int tc_launch(const Device *dev, const PagedAttn &p, int units, cudaStream_t st) {
    using S = TcShape<KB, WIDE>;
    static DeviceOnce once;
    if (once.first(dev->ordinal)) IM_CUDA_CHECK(cudaFuncSetAttribute((paged_tc_kernel<BF16, KB, WIDE>), cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    IM_CUDA_CHECK(launch_k(paged_tc_kernel<BF16, KB, WIDE>, dim3(p.ctas), dim3(kTcThreads), (size_t)S::kSmem, st, p, units, dev->err_flag));
    const long long rows = std::min<long long>(S::kRows, (long long)p.max_new * p.group);
    IM_CUDA_CHECK(launch_k(paged_tc_join_kernel<BF16, KB, WIDE>, dim3((unsigned)(units * p.kv.nkv), (unsigned)((rows + 31) / 32 * (16 * KB) / (kTcJoinThreads / 32))),
                           dim3(kTcJoinThreads), 0, st, p));
    return IM_OK;
}

}  // namespace

int paged_tc_rows(int hd, long long rows) {
    if (hd != 64 && hd != 128) return 0;
    return rows <= 16 ? 0 : rows <= 128 ? 128 : 256;
}

int paged_tc_launch(const Device *dev, const PagedAttn &p, bool bf16, int rows, int units, cudaStream_t st) {
    const bool wide = rows == 256;
#define IM_RUN(B, KB) (wide ? tc_launch<B, KB, true>(dev, p, units, st) : tc_launch<B, KB, false>(dev, p, units, st))
    if (p.kv.hd == 64) return bf16 ? IM_RUN(true, 1) : IM_RUN(false, 1);
    return bf16 ? IM_RUN(true, 2) : IM_RUN(false, 2);
#undef IM_RUN
}

}  // namespace im
