// Attention that also adds up what every position of the cache is worth to the call's tokens: the sums by which an eviction chooses (paged_evict.cu).
//
//   out[t, h] = sum_j p_thj v_j,   sum[s, g, j] += sum over the new tokens t of s and the heads h of KV head g of p_thj,   p = softmax as in paged_attn.cu
//
// A weight is known once its row's maximum and sum over all positions are: the attention kernels leave both for every row, and a second look at the scores
// follows. Up to 16 rows of a KV head (single tokens) the scores themselves are kept, 4 bytes a row and position against 4 * head_dim of keys
// and values, and a position's thread adds up its rows' weights; short contexts do it in the attention's own launch. With more rows keeping the scores would
// cost more than the keys: the tensor cores compute them again, transposed: positions in the lanes of tensor memory, query rows in its columns, so that a position
// is one thread's. No atomics, and the same sums on every run.
//
// 32 sequences of up to 8192 rows, a token each (589 MB): 124 us, of which the attention 107 (105 without the scores) and the sums with the join 14 (24 with a position a thread and the join by
// itself). The last 64 tokens of 32001 rows (256 rows of a KV head): 90 us, of which the attention 45 and the sums 33: 6 until the first scores, then a tile of 128 positions and 256 rows every 2 us
// (mma.sync in place of tcgen05: 134).
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "paged_tc.cuh"

namespace im {
namespace {

constexpr int kSumThreads = 256, kSumWarps = kSumThreads / 32, kSumPositions = 4 * kSumThreads;

// Behind attention in shares, in one launch: blocks below `joins` join the outputs of items that a cut divides, eight rows each, the others add up the weights of an item, four positions a
// thread. Both find the rows' maxima and sums in the parts.
template <bool BF16, int HD>
__global__ void __launch_bounds__(kSumThreads) paged_sum_kernel(const __grid_constant__ PagedAttn p, int joins, int row_blocks, int chunks) {
    constexpr int R = 16;
    __shared__ float norms[R];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if ((int)blockIdx.x < joins) {
        join_row<BF16, R, HD>(p, blockIdx.x / row_blocks, (blockIdx.x % row_blocks) * kSumWarps + warp);
        return;
    }
    const int item = (blockIdx.x - joins) / chunks, unit = item / p.kv.nkv, head = item - unit * p.kv.nkv, chunk = (blockIdx.x - joins) % chunks;
    const PagedUnit u = paged_unit<R, kWeigh>(p, unit);
    if ((long long)chunk * kSumPositions >= u.end) return;
    const int2 span = *reinterpret_cast<const int2 *>(p.spans + 2 * (long long)item);
    for (int r = warp; r < u.rows; r += kSumWarps) {
        float2 ml;
        if (span.x < 0) {
            ml = p.stat[(long long)item * R + r];
        } else {
            ml = row_parts(p.part_ml, span, R, r, lane, 32);
            const float top = warp_max(ml.x);
            ml = make_float2(top, warp_sum(ml.x == -INFINITY && ml.y == 0.0f ? 0.0f : ml.y * ex2(ml.x - top)));
        }
        if (lane == 0) norms[r] = row_norm(ml);
    }
    __syncthreads();
    const float *scores = p.scores + (long long)item * p.score_rows * p.score_cap;
    float *sums = p.sums + u.seq * p.sum_seq + head * p.sum_head;
    const bool aligned = reinterpret_cast<uintptr_t>(sums) % 16 == 0;
    for (long long at = (long long)chunk * kSumPositions + 4 * tid; at < u.end; at += (long long)chunks * kSumPositions) {
        const int pos = (int)at;
        if (at + 4 <= p.score_cap) {  // (a multiple of 64)
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (int r = 0; r < u.rows; r++) {
                const float4 s = *reinterpret_cast<const float4 *>(scores + (long long)r * p.score_cap + pos);
                v.x += ex2(s.x + norms[r]); v.y += ex2(s.y + norms[r]); v.z += ex2(s.z + norms[r]); v.w += ex2(s.w + norms[r]);
            }
            const float all = (v.x + v.y) + (v.z + v.w);
            if (all == all && aligned && pos + 4 <= min(u.len, p.sum_cols)) {
                float4 *to = reinterpret_cast<float4 *>(sums + pos);
                const float4 o = *to;
                *to = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
            } else {
                const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (pos + j < u.end) add_sum(p, u, head, pos + j, seen_sum<BF16, HD>(p, u, head, pos + j, norms, x[j]));
            }
        } else {
            for (int j = 0; j < 4 && at + j < u.end; j++) add_sum(p, u, head, pos + j, plain_sum<BF16, HD>(p, u, head, pos + j, norms));
        }
    }
}

// Sums from queries and keys on tcgen05, one CTA per SM, an equal share of the list of all (sequence, KV head) items' tiles of 128 positions. Up to
// kBlockRows of an item's rows stay in shared memory while its tiles of keys pass (more: once more, block by block):
//     S^T = K Q^T    128 positions x up to 256 rows, f32 in tensor memory, two buffers
//     sum += 2^(scale S^T + norm of the row), a position per thread, two sets of four warps, every other tile each
// What bounds it: a tile of 256 rows is 2048 clocks of exponentials (16 a clock and SM), 1024 of products and takes 3600; 32 columns of a warp take 740 clocks where two warps of a
// scheduler need 512 for their exponentials. Exponentials by polynomials for three of eight columns changed nothing; nor did two loads of scores at a time.
// All waits are bounded: one that runs out sets the device error word, every warp then runs to its end.
template <int KB>
struct WeighShape {
    static constexpr int kBlockRows = KB == 4 ? 128 : 256;
    static constexpr int kBlock = 128 * 128, kSlot = KB * kBlock;  // bytes of 128 positions of 64 columns, of a tile of keys
    static constexpr int kQBlock = kBlockRows * 128, kQ = KB * kQBlock;
    static constexpr int kK = KB == 4 ? 2 : KB == 2 ? 4 : 6;       // tiles of keys
    static constexpr int kBars = 2 * kK + 2 + 4;
    static constexpr int kSmall = 8 * 16 + kBlockRows * 4 + kTcCopyWarps * 32 * 8 + kBars * 8 + 16;  // presence bits, norms, offsets, barriers, address
    static constexpr int kTiles = kQ + kK * kSlot;
    static constexpr int kSmem = (kSmall + 1023) / 1024 * 1024 + kTiles;
    static_assert(kSmem <= 232448, "shared memory of an SM");
};
constexpr int kAllRows = 1 << 30;  // a unit is a sequence

// Bit j: row `row` + j of a sequence (token, query head) sees position pos.
__device__ __forceinline__ uint32_t rows_seeing(const PagedAttn &p, const PagedUnit &u, int row, int pos) {
    const int d = pos - u.len, n = u.rows - row;  // place among the new rows
    const uint32_t are = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1;
    if (pos >= u.end || d >= u.fresh) return 0u;
    if (d < 0) return are;
    if (!p.mask) {  // those of the d-th token and of later ones
        const long long from = (long long)d * p.group - row;
        return from <= 0 ? are : from >= 32 ? 0u : are & ~((1u << from) - 1);
    }
    if (d >= 64 * p.mask_words) return 0u;
    uint32_t seen = 0;
    int t = row / p.group, left = p.group - (row - t * p.group);  // rows of token t from here on
    const uint64_t *word = p.mask + (long long)(u.tok0 + t) * p.mask_words + (d >> 6);
#pragma unroll 1
    for (int j = 0; j < 32 && j < n; word += p.mask_words, left = p.group) {
        const int m = min(left, 32 - j);
        if (__ldg(word) >> (d & 63) & 1) seen |= (m == 32 ? 0xffffffffu : (1u << m) - 1) << j;
        j += m;
    }
    return seen & are;
}

template <bool BF16, int KB>
__global__ void __launch_bounds__(kTcThreads, 1) paged_weigh_kernel(const __grid_constant__ PagedAttn p, int units, int stat_rows, int stat_tiles, const float2 *parts, int *err) {
    using S = WeighShape<KB>;
    constexpr int HD = 64 * KB, SK = S::kK, BR = S::kBlockRows;
    extern __shared__ __align__(16) unsigned char weigh_smem[];
    uint32_t *there = reinterpret_cast<uint32_t *>(weigh_smem);               // [8 tiles][4]: bit j of word w: row 32 w + j of the tile is in the cache
    float *norms = reinterpret_cast<float *>(there + 32);                     // [BR]
    long long *offs = reinterpret_cast<long long *>(norms + BR);              // [copying warps][32]
    uint64_t *kfull = reinterpret_cast<uint64_t *>(offs + kTcCopyWarps * 32), *kempty = kfull + SK, *qfull = kempty + SK, *qempty = qfull + 1, *sfull = qempty + 1, *sempty = sfull + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sempty + 2);
    unsigned char *Qs = weigh_smem + (S::kSmem - S::kTiles), *Ks = Qs + S::kQ;
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
        mbar_init(qfull, kTcCopyWarps * 32);
        mbar_init(qempty, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sfull[i], 1);
            mbar_init(&sempty[i], 4);
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
    pdl_trigger();
    if (!p.early) pdl_wait();
    PagedUnit at;
    const Share share = units <= 32 ? warp_share<kAllRows, kTcTile, kWeigh>(p, units, p.ctas, at) : find_share<kAllRows, kTcTile, kTcThreads, kWeigh>(p, units, p.ctas, reinterpret_cast<long long *>(Qs), at);
    Items<kAllRows, kWeigh> it(p, units, share, at);
    bool ok = true;
    int block = 0;  // blocks of rows so far
    auto columns = [&](const PagedUnit &u, int row0) { return min((u.rows - row0 + 31) / 32 * 32, BR); };
    if (warp >= kTcCopy) {
        // ---- copies
        const int w0 = (warp - kTcCopy) * 32;
        long long *mine = offs + w0;
        auto room = [&](uint64_t *bar, uint32_t parity) {
            if (ok && !mbar_try_wait(bar, parity)) ok = wait_for(bar, parity, err);
            __syncwarp();
        };
        auto requested = [&](uint64_t *bar) {
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
        };
        // 32 rows, the first at dst, whose offsets (elements from base; -1: none) lanes name; blocks of 64 columns `apart` bytes from one another
        auto rows32 = [&](unsigned char *dst, int apart, const uint16_t *base, long long o) {
            constexpr int CH = 8 * KB, RPI = 32 / CH > 0 ? 32 / CH : 1;
            __syncwarp();
            mine[lane] = o;
            __syncwarp();
            const int c = lane % CH, r0 = lane / CH;
            const uint32_t to = smem_u32(dst) + (c >> 3) * apart + r0 * 128;
#pragma unroll 1
            for (int i0 = 0; i0 < 32 / RPI; i0 += 8) {
                long long x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = mine[(i0 + i) * RPI + r0];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int r = (i0 + i) * RPI;
                    cp16(to + r * 128 + (((c & 7) ^ ((r + r0) & 7)) << 4), base + (x[i] < 0 ? 0 : x[i] + c * 8), x[i] >= 0);
                }
            }
        };
        int kc = 0;
        auto lookup = [&](const PagedUnit &u, int head, int pos) -> long long {
            if (pos >= u.end) return -1;
            const long long o = p.kv.row_of(u.seq, pos);
            return o < 0 ? -1 : o + (long long)head * p.kv.page * HD;
        };
        while (it.next()) {
            const PagedUnit &u = it.u;
            for (int row0 = 0; row0 < u.rows; row0 += BR, block++) {
                long long o = lookup(u, it.head, it.t0 * kTcTile + w0 + lane);
                if (block > 0) room(qempty, (block - 1) & 1);
                const int n = columns(u, row0);
                for (int r = w0; r < n; r += kTcCopyWarps * 32) {
                    const int row = row0 + r + lane, t = row / p.group, g = row - t * p.group;
                    const bool is = row < u.rows;
                    rows32(Qs + r * 128, S::kQBlock, p.q, is ? (u.tok0 + t) * p.qs + (long long)(it.head * p.group + g) * HD : -1);
                }
                requested(qfull);
                for (int t = it.t0; t < it.t1; t++) {
                    const int ks = kc % SK;
                    const long long next = t + 1 < it.t1 ? lookup(u, it.head, (t + 1) * kTcTile + w0 + lane) : -1;
                    if (kc >= SK) room(&kempty[ks], (kc / SK - 1) & 1);
                    const unsigned word = __ballot_sync(0xffffffffu, o >= 0);
                    if (lane == 0) {
                        there[(kc & 7) * 4 + w0 / 32] = word;
                        mbar_arrive(&kfull[ks]);
                    }
                    rows32(Ks + ks * S::kSlot + w0 * 128, S::kBlock, p.kc, o);
                    requested(&kfull[ks]);
                    kc++;
                    o = next;
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == kTcMma) {
        // ---- products; instruction descriptor as in paged_attn_tc.cu, N (rows) in bits 17-22
        constexpr uint32_t kType = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(128 >> 4) << 24);
        const uint32_t one = elected();
        const uint64_t qd = desc_sw128(smem_u32(Qs), 16), kd = desc_sw128(smem_u32(Ks), 16);
        int ks = 0, tile = 0;
        uint32_t kturn = 0;
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            if (ok && !mbar_try_wait(bar, parity)) ok = wait_for(bar, parity, err);
            __syncwarp();
        };
        while (it.next()) {
            for (int row0 = 0; row0 < it.u.rows; row0 += BR, block++) {
                const uint32_t idesc = kType | (uniform(columns(it.u, row0)) >> 3 << 17);
                wait(qfull, block & 1);
#pragma unroll 1
                for (int t = it.t0; t < it.t1; t++, tile++) {
                    wait(&kfull[ks], kturn);
                    if (tile >= 2) wait(&sempty[tile & 1], (tile / 2 - 1) & 1);
                    copies_landed();
                    fence_after();
                    if (ok) {
                        const uint64_t a = kd + ks * (S::kSlot / 16);
#pragma unroll
                        for (int j = 0; j < KB * 4; j++)
                            umma_ss(one, tmem + (uint32_t)((tile & 1) * 256), a + (j / 4 * S::kBlock + (j & 3) * 32) / 16, qd + (j / 4 * S::kQBlock + (j & 3) * 32) / 16, idesc, j > 0);
                        umma_commit(one, &sfull[tile & 1]);
                        umma_commit(one, &kempty[ks]);
                        if (t == it.t1 - 1) umma_commit(one, qempty);
                    }
                    if (++ks == SK) ks = 0, kturn ^= 1;
                }
            }
        }
        __syncwarp();
    } else {
        // ---- sums: a position per thread
        const int h = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(h * 256);
        const uint64_t scale_two = two(p.scale2, p.scale2);
        int tile = 0;
        while (it.next()) {
            const PagedUnit &u = it.u;
            for (int row0 = 0; row0 < u.rows; row0 += BR, block++) {
                const int n = columns(u, row0);
                both_halves();  // the norms before have been read
                if (tid < n) {
                    const int row = row0 + tid;
                    float2 ml = make_float2(-INFINITY, 0.0f);
                    if (row < u.rows) {
                        const int tile = row / stat_rows, r = row - tile * stat_rows;
                        const long long item = ((long long)u.seq * stat_tiles + tile) * p.kv.nkv + it.head;
                        const int2 span = parts ? *reinterpret_cast<const int2 *>(p.spans + 2 * item) : make_int2(-1, 0);
                        ml = span.x < 0 ? p.stat[item * stat_rows + r] : row_parts(parts, span, stat_rows, r, 0, 1);
                    }
                    norms[tid] = row_norm(ml);
                }
                both_halves();
                for (int t = it.t0; t < it.t1; t++, tile++) {
                    if ((tile & 1) != h) continue;
                    if (ok && !wait_for(&sfull[h], (tile / 2) & 1, err)) ok = false;
                    fence_after();
                    const int pos = t * kTcTile + r;
                    const bool is = (there[(tile & 7) * 4 + (warp & 3)] >> lane & 1u) != 0;
                    const bool edge = t * kTcTile + kTcTile > u.len;  // some row may not see some position
                    uint64_t sum[2] = {0, 0};
                    auto add = [&](uint32_t *s, int c) {  // 32 columns
                        if (edge) {
                            const uint32_t seen = rows_seeing(p, u, row0 + c, pos);
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (!(seen >> j & 1u)) s[j] = p.scale2 < 0.0f ? 0x7f800000u : 0xff800000u;  // a score of -inf
                        }
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const float4 a = *reinterpret_cast<const float4 *>(norms + c + 4 * j);
                            const uint64_t x0 = fma_two(two(__uint_as_float(s[4 * j]), __uint_as_float(s[4 * j + 1])), scale_two, two(a.x, a.y));
                            const uint64_t x1 = fma_two(two(__uint_as_float(s[4 * j + 2]), __uint_as_float(s[4 * j + 3])), scale_two, two(a.z, a.w));
                            const float2 e0 = of_two(x0), e1 = of_two(x1);
                            sum[0] = add_two(sum[0], two(ex2(e0.x), ex2(e0.y)));
                            sum[1] = add_two(sum[1], two(ex2(e1.x), ex2(e1.y)));
                        }
                    };
                    uint32_t s0[32], s1[32];  // the next columns are on their way while these are added
                    ld32(ts, s0);
#pragma unroll 1
                    for (int c = 0; c < n; c += 64) {
                        tmem_wait_ld();
                        if (c + 32 < n) ld32(ts + (uint32_t)(c + 32), s1);
                        add(s0, c);
                        if (c + 32 >= n) break;
                        tmem_wait_ld();
                        if (c + 64 < n) ld32(ts + (uint32_t)(c + 64), s0);
                        add(s1, c + 32);
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sempty[h]);
                    const float2 x = of_two(sum[0]), y = of_two(sum[1]);
                    float v = (x.x + x.y) + (y.x + y.y);
                    // an infinite or missing key times the zeros that fill up the rows, or something that is one: from the rows that see it alone
                    if (__any_sync(0xffffffffu, is && !(v - v == 0.0f))) {
                        PagedUnit part = u;
                        part.row0 = row0;
                        part.rows = min(u.rows - row0, BR);
                        const float w = plain_sum<BF16, HD>(p, part, it.head, pos, norms);
                        if (!(v - v == 0.0f)) v = w;
                    }
                    if (pos < u.end) add_sum(p, u, it.head, pos, is ? v : 0.0f, row0 == 0);
                }
            }
        }
    }
    fence_before();
    sync_and_settle(ok);
    if (p.early && blockIdx.x == 0) pdl_wait();  // this launch ends after the one before it
    if (warp == kTcMma) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Room for scores: where there are up to 16 rows of a KV head and 256 MB hold them (32 sequences of 32 heads: 65536 positions).
constexpr size_t kScoreMost = (size_t)256 << 20;
struct WeighPlan {
    AttnPlan attn;
    int cap, rows;        // positions and rows of an item's scores, 0: none are kept
    size_t attn_bytes, stat_bytes, score_bytes;
    size_t used, bytes;   // by a call of this length, by any up to it
};
WeighPlan weigh_plan(const Device *dev, const PagedView &v, int group, int max_new, int max_len) {
    WeighPlan a;
    a.attn = attn_plan(dev, v.nseq, v.nkv, v.hd, group, max_new, max_len);
    const size_t items = (size_t)a.attn.units * v.nkv;
    a.attn_bytes = (a.attn.bytes + 15) / 16 * 16;
    a.stat_bytes = (items + (a.attn.rows > 16 ? 2 * (size_t)a.attn.ctas : 0)) * a.attn.rows * 8;
    a.rows = group * max_new;
    a.cap = 0;
    size_t most = 0;
    if (a.attn.rows == 16 && a.attn.row_tiles == 1 && items > 0) {
        const size_t of_tile = items * a.rows * 4 * 64, tiles = ((size_t)max_len + 63) / 64;
        most = std::min(tiles, kScoreMost / of_tile) * of_tile;
        if (tiles * of_tile <= kScoreMost) a.cap = (int)std::min<size_t>(tiles * 64, INT_MAX / 64 * 64);
    }
    a.score_bytes = a.cap ? most : 0;
    a.used = a.attn_bytes + a.stat_bytes + a.score_bytes;
    a.bytes = a.attn_bytes + a.stat_bytes + most;
    return a;
}

template <bool BF16, int HD>
int sums(const Device *dev, const PagedAttn &p, const WeighPlan &plan, int max_len, cudaStream_t st) {
    if (p.scores) {
        const long long items = (long long)plan.attn.units * p.kv.nkv, row_blocks = (plan.rows + kSumWarps - 1) / kSumWarps;
        const long long chunks = std::max(1ll, std::min<long long>((max_len + (long long)kSumPositions - 1) / kSumPositions, (1ll << 30) / items));
        IM_CUDA_CHECK(launch_k(paged_sum_kernel<BF16, HD>, dim3((unsigned)(items * (row_blocks + chunks))), dim3(kSumThreads), 0, st, p, (int)(items * row_blocks), (int)row_blocks, (int)chunks));
        return IM_OK;
    }
    using S = WeighShape<HD / 64>;
    static DeviceOnce once;
    if (once.first(dev->ordinal)) IM_CUDA_CHECK(cudaFuncSetAttribute((paged_weigh_kernel<BF16, HD / 64>), cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    PagedAttn w = p;
    w.row_tiles = 1;
    w.early = plan.attn.rows > 16;  // the join in front of it triggers it once the attention is done
    w.ctas = (int)std::max(1ll, std::min<long long>(dev->sm_count, (long long)p.kv.nseq * p.kv.nkv * ((max_len + (long long)kTcTile - 1) / kTcTile)));
    IM_CUDA_CHECK(launch_k(paged_weigh_kernel<BF16, HD / 64>, dim3(w.ctas), dim3(kTcThreads), (size_t)S::kSmem, st, w, p.kv.nseq, plan.attn.rows, plan.attn.row_tiles,
                           plan.attn.cluster ? nullptr : plan.attn.rows > 16 ? p.stat_parts : p.part_ml, dev->err_flag));
    return IM_OK;
}

}  // namespace
}  // namespace im

IM_EXPORT size_t im_cuda_paged_attention_weights_scratch_bytes(const im_device *dev, const im_paged_kv *kv, int num_heads, int max_new, int max_len) {
    try {
        im::PagedView v;
        if (!dev || im::paged_view(kv, 0, &v) != IM_OK || im::attn_check(kv, num_heads, max_new) != IM_OK || max_len < 0) return 0;
        return im::weigh_plan(dev, v, num_heads / v.nkv, max_new, im::attn_length(v, max_len)).bytes;
    } catch (...) {
        return 0;
    }
}

IM_EXPORT int im_cuda_paged_attention_weights(im_device *dev, const im_paged_kv *kv, const im_paged_weights_args *args, void *stream) {
    IM_GUARD_BEGIN
    using namespace im;
    PagedAttn p;
    bool empty;
    IM_REQUIRE(kv && args && kv->num_kv_heads > 0, "kv or args is NULL, or there are no heads");
    const im_paged_attention_args &x = args->attention;
    const int rows = args->rows;
    const int64_t seq_stride = args->seq_stride, head_stride = args->head_stride;
    float *const weights_dev = args->weights_dev;
    const int64_t most = (int64_t)1 << 40;
    IM_REQUIRE(rows >= 1 && head_stride >= rows && seq_stride <= most / std::max(kv->num_seqs, 1) && head_stride <= most / kv->num_kv_heads &&
                   (kv->num_seqs <= 1 || seq_stride >= (kv->num_kv_heads - 1) * head_stride + rows),
               "sums of different sequences and heads overlap");
    if (x.num_tokens > 0 && kv->num_seqs > 0) {
        IM_REQUIRE(weights_dev && reinterpret_cast<uintptr_t>(weights_dev) % 4 == 0, "the sums are NULL or not 4-byte aligned");
        const long long span = 4 * ((kv->num_seqs - 1) * (long long)seq_stride + (kv->num_kv_heads - 1) * head_stride + rows), row = 2ll * x.num_heads * kv->head_dim;
        IM_REQUIRE(!share_memory(weights_dev, span, x.q_dev, 2 * (x.num_tokens - 1) * (long long)x.q_stride + row) && !share_memory(weights_dev, span, x.out_dev, 2 * (x.num_tokens - 1) * (long long)x.out_stride + row),
                   "the sums lie over the queries or the outputs");
        PagedView v;
        const int rc = paged_view(kv, x.layer, &v);
        if (rc != IM_OK) return rc;
        IM_REQUIRE(!share_memory(weights_dev, span, v.table, 4 * ((v.nseq - 1) * v.table_stride + v.width)) && !share_memory(weights_dev, span, v.len, 4ll * v.nseq) &&
                       !share_memory(weights_dev, span, x.token_start_dev, 4ll * (v.nseq + 1)) && (!x.mask_dev || !share_memory(weights_dev, span, x.mask_dev, 8ll * x.num_tokens * x.mask_words)),
                   "the sums lie over the page table, the lengths, the tokens' starts or the mask");
    }
    int rc = attn_args(dev, kv, x.layer, x.q_dev, x.q_stride, x.out_dev, x.out_stride, x.num_heads, x.token_start_dev, x.num_tokens, x.max_new, x.mask_dev, x.mask_words, x.scale, x.max_len, &p,
                       &empty);
    if (rc != IM_OK || empty) return rc;
    const int max_len = attn_length(p.kv, x.max_len);
    const WeighPlan plan = weigh_plan(dev, p.kv, p.group, x.max_new, max_len);
    IM_REQUIRE(plan.used == 0 || (x.scratch_dev && aligned16(x.scratch_dev) && x.scratch_bytes >= plan.used), "paged attention with sums needs %zu bytes of 16-byte aligned scratch (got %zu)",
               plan.used, x.scratch_dev ? x.scratch_bytes : (size_t)0);
    attn_lay_out(&p, plan.attn, max_len, x.scratch_dev);
    unsigned char *at = static_cast<unsigned char *>(x.scratch_dev) + plan.attn_bytes;
    p.stat = reinterpret_cast<float2 *>(at);
    p.stat_parts = p.stat + (size_t)plan.attn.units * p.kv.nkv * plan.attn.rows;
    p.scores = plan.cap ? reinterpret_cast<float *>(at + plan.stat_bytes) : nullptr;
    p.score_cap = plan.cap;
    p.score_rows = plan.rows;
    p.sums = weights_dev;
    p.sum_seq = seq_stride;
    p.sum_head = head_stride;
    p.sum_cols = rows;
    const cudaStream_t st = as_stream(stream);
    const bool bf16 = kv->dtype == IM_DTYPE_BF16;
    rc = plan.attn.rows >= 128 ? paged_tc_weigh_launch(dev, p, bf16, plan.attn.rows, plan.attn.units, st) : paged_weigh_launch(dev, p, bf16, plan.attn.units, plan.attn.cluster, !p.scores, st);
    if (rc != IM_OK || (plan.attn.cluster && p.scores)) return rc;
#define IM_RUN(HD) (bf16 ? sums<true, HD>(dev, p, plan, max_len, st) : sums<false, HD>(dev, p, plan, max_len, st))
    switch (kv->head_dim) {
    case 64: return IM_RUN(64);
    case 128: return IM_RUN(128);
    default: return IM_RUN(256);
    }
#undef IM_RUN
    IM_GUARD_END
}
