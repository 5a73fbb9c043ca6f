// paged_wide_sm100.cuh -- paged_decode for many query heads per K/V head, on
// the tcgen05 tensor cores.
//
// With G query heads sharing a K/V head, a byte of 16-bit K or V meets 2 G
// operations (3 G with P in two parts): from about G = 16 on the warp MMAs of
// paged_sm100.cuh cannot keep up with the memory any more.  Here the query
// heads are the rows of a 128-row tile and a step is 128 keys: S = Q K^T
// (128 x 128) and O += P V (128 x D), with Q, S, P and O in tensor memory.
//
// A lane of tensor memory is reached by one warp of four only, so 32 query
// heads alone would leave the softmax to one of the SM's four schedulers.  The
// tile therefore holds kCopies copies of the heads (4 of 32, 2 of 64, 1 of 128):
// every copy gets all the scores, but its warps take the softmax of their
// 128 / kCopies keys only, and P V of those keys adds to that copy's rows only
// (the others are disabled lanes of the MMA).  The copies are states of their own,
// joined when an item ends, as the parts of different CTAs are.
//
//   warps 0-3  softmax: lanes 32 w ..
//   warp 4     allocates tensor memory and issues Q K^T
//   warp 5     issues P V (one warp for both held a step for 2100 cycles)
//   warps 6 .. producers: page look-ups, and 16-byte asynchronous copies of
//              whole rows into a ring of units (128 rows of K or of V, swizzled
//              as the MMA descriptors want them)
//
// A step's 128 keys are 64 KB of K and V at head_dim 128: 1.4 us at the memory's rate, in
// which the SM issues 8 + 16 MMAs and the softmax takes about 1000 cycles.  Measured (batch 16,
// 4 K/V heads, 8192 keys, bf16): 32 query heads each, head_dim 128 59 us (4.5 TB/s; the warp
// MMAs 86.5), 64 heads 67 us (153), head_dim 64 43 us (57); 3 requests of up to 131072 keys with
// one K/V head 41 us, of which 17 us stream at the memory's rate and the rest is latency.
//
// S is double buffered: Q K^T of step j + 1 runs while the softmax works on
// step j.  P's high and low parts replace a warp's own scores.  One CTA per SM.
//
// Every mbarrier wait is bounded.  On expiry the waiter records itself in
// g_paged_status and raises the CTA's abort flag; the roles leave their loops,
// copies and MMAs in flight are waited for, tensor memory is freed.  The softmax
// warps' hardware barriers have no limit of their own: see softmax_together.
#pragma once
#include "paged_sm100.cuh"

namespace nczp {

constexpr unsigned long long kPagedWaitLimit = 4000000000ull;  // SM cycles, about 2 s
__device__ uint32_t g_paged_status = 0u;
__device__ unsigned long long g_paged_wait_limit = kPagedWaitLimit;
__device__ int g_paged_test_drop = 0;   // test hook: the first step's scores are never announced
__device__ int g_paged_test_leave = 0;  // test hook: a softmax warp gives up where the first item ends

// Where a bounded wait gave up (bits 24.. of the status word).
enum : uint32_t {
    kSiteEmpty = 1, kSiteFull, kSiteQFull, kSiteScores, kSiteP, kSiteOFree, kSiteODone, kSiteMerge, kSiteDrain
};

constexpr int kScoreWarp = 4, kValueWarp = 5, kProducerWarp = 6;
constexpr int kProducers = 4;  // warps that fill a unit, 32 rows each
constexpr int kWideTile = 128;  // keys per step
constexpr int kMaskRing = 16;   // steps whose masks are kept; producers run at most 7 steps ahead
constexpr int kMergeStride = 20;  // floats of a row's 16 columns in the merge buffer

// D = 64 or 128; kQRows = 32, 64 or 128 query heads per item.
template <int D_, bool kBf16_, int kQRows_>
struct Wide {
    static constexpr int D = D_, kQRows = kQRows_;
    static constexpr bool kBf16 = kBf16_;
    static constexpr int kCopies = 128 / kQRows;        // of the query heads
    static constexpr int kCols = kWideTile / kCopies;   // keys of a softmax warp
    static constexpr int kPanels = D / 64;              // 64-element (128-byte) panels of a row
    static constexpr int kPanel = kWideTile * 128;      // bytes of a panel of a unit
    static constexpr int kUnit = kPanels * kPanel;
    static constexpr int kMerge = kCopies > 1 ? 2 * 128 * kMergeStride * 4 : 0;
    static constexpr int kFit = (227 * 1024 - 4096 - kMerge) / kUnit;
    static constexpr int kUnits = kFit < 12 ? kFit : 12;
    // With 32 query heads the softmax warps leave registers for four producer warps for K and four
    // for V; else four take both in turn.
    static constexpr int kTeams = kCopies == 4 ? 2 : 1;
    static constexpr int kThreads = (kProducerWarp + kTeams * kProducers) * 32;
    // Units a producer warp has on their way: 128 KB over the CTA, a unit less than it has slots.
    static constexpr int kSlots = kUnits / kTeams;
    static constexpr int kDepth = 131072 / kUnit / kTeams < kSlots - 1 ? 131072 / kUnit / kTeams : kSlots - 1;
    static_assert(kUnits % kTeams == 0 && kDepth >= 2, "");
    static constexpr int kSmem = 1024 + kUnits * kUnit + kMerge;
    // A producer warp's 32 rows of a unit: 16-byte chunks, rows per copy instruction, instructions.
    static constexpr int kChunks = D / 8, kRowsPerCopy = 32 / kChunks, kRowCopies = 32 / kRowsPerCopy;
};

// A wait by parity tells a phase from its neighbours only, so a barrier's waiter
// must be within one phase of it: what belongs to a step has a barrier per score
// buffer, whose next phase cannot come before the step that waits.
struct WideBars {
    uint64_t full[12], empty[12], q_full[2], s_full[2], p_full[2], o_done[2], o_free, drain[2];
};

__device__ __forceinline__ void paged_give_up(volatile uint32_t *abort_flag, uint32_t site) {
    *abort_flag = 1u;
    atomicCAS(&g_paged_status, 0u, 0x80000000u | (site << 24) | (blockIdx.x & 0xFFFFFFu));
}
__device__ __noinline__ bool paged_wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag,
                                             uint32_t site, bool honor_abort) {
    const unsigned long long t0 = ncz::sm_clock();
    for (uint32_t it = 1;; ++it) {
        if (ncz::mbar_try_wait(bar, parity)) return true;
        if ((it & 15u) == 0u) {
            if (honor_abort && *abort_flag) return false;
            if (ncz::sm_clock() - t0 > g_paged_wait_limit) {
                paged_give_up(abort_flag, site);
                return false;
            }
        }
    }
}
// All lanes wait; the answer is the same in all of them.
__device__ __forceinline__ bool paged_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *abort_flag,
                                           uint32_t site, bool honor_abort = true) {
    const uint32_t b = smem_u32(bar);
    const bool ok = ncz::mbar_try_wait(b, parity) || paged_wait_slow(b, parity, abort_flag, site, honor_abort);
    return __all_sync(~0u, ok);
}

// O (+)= P V for 16 kSteps keys, high and then low parts of P (8 columns of
// `high` and `low` per 16 keys), on the lanes whose bits in m0 .. m3 are 0.  The
// whole converged warp executes it and one lane issues; `accumulate` applies to
// the first MMA, the others always do.  One block for all of them: issued one by
// one, 16 MMAs kept the issuing warp for 750 cycles of a step.
template <int kSteps>
__device__ __forceinline__ void umma_ts_lanes(uint32_t d, uint32_t high, uint32_t low, uint64_t b_desc, uint64_t b_step,
                                              uint32_t idesc, uint32_t accumulate, uint32_t m0, uint32_t m1,
                                              uint32_t m2, uint32_t m3) {
    static_assert(kSteps == 2 || kSteps == 4, "key steps");
    if constexpr (kSteps == 2) {
        asm volatile(
            "{\n.reg .pred p, e;\nelect.sync _|e, -1;\nsetp.ne.b32 p, %2, 0;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%7], %8, %1, {%3, %4, %5, %6}, p;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%9], %10, %1, {%3, %4, %5, %6}, 1;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%11], %8, %1, {%3, %4, %5, %6}, 1;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%12], %10, %1, {%3, %4, %5, %6}, 1;\n}\n" ::"r"(d),
            "r"(idesc), "r"(accumulate), "r"(m0), "r"(m1), "r"(m2), "r"(m3), "r"(high), "l"(b_desc), "r"(high + 8),
            "l"(b_desc + b_step), "r"(low), "r"(low + 8)
            : "memory");
    } else {
        asm volatile(
            "{\n.reg .pred p, e;\nelect.sync _|e, -1;\nsetp.ne.b32 p, %2, 0;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%7], %8, %1, {%3, %4, %5, %6}, p;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%9], %10, %1, {%3, %4, %5, %6}, 1;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%11], %12, %1, {%3, %4, %5, %6}, 1;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%13], %14, %1, {%3, %4, %5, %6}, 1;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%15], %8, %1, {%3, %4, %5, %6}, 1;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%16], %10, %1, {%3, %4, %5, %6}, 1;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%17], %12, %1, {%3, %4, %5, %6}, 1;\n"
            "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%18], %14, %1, {%3, %4, %5, %6}, 1;\n}\n" ::"r"(d),
            "r"(idesc), "r"(accumulate), "r"(m0), "r"(m1), "r"(m2), "r"(m3), "r"(high), "l"(b_desc), "r"(high + 8),
            "l"(b_desc + b_step), "r"(high + 16), "l"(b_desc + 2 * b_step), "r"(high + 24), "l"(b_desc + 3 * b_step),
            "r"(low), "r"(low + 8), "r"(low + 16), "r"(low + 24)
            : "memory");
    }
}

// Hardware barriers of the four softmax warps.
//
// softmax_together: whether all four come with `ok`.  Each warp calls it once for every
// item that it ends, or, where one of its waits ran out first, once with false as it leaves,
// so all four are in the same call; a warp that hears false leaves and calls no barrier
// again.  Between two calls a warp waits at limited waits only, hence every call ends.
// softmax_sync: only between a call that said true and the end of that item, where no warp can leave.
__device__ __forceinline__ bool softmax_together(bool ok) {
    uint32_t all;
    asm volatile(
        "{\n.reg .pred mine, all;\nsetp.ne.b32 mine, %1, 0;\nbar.red.and.pred all, 1, 128, mine;\n"
        "selp.b32 %0, 1, 0, all;\n}\n"
        : "=r"(all)
        : "r"(ok ? 1u : 0u)
        : "memory");
    return all != 0;
}
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <class T>
__global__ void __launch_bounds__(T::kThreads, 1) paged_decode_wide(const DecodeParams p) {
    constexpr int D = T::D, kCopies = T::kCopies, kCols = T::kCols, kPairs = kCols / 2;
    constexpr bool kBf16 = T::kBf16;
    using ncz::mbar_arrive;
    extern __shared__ char smem_raw[];
    __shared__ WideBars bars;
    __shared__ uint32_t s_mask[kMaskRing][4];
    __shared__ float2 s_ml[128];
    __shared__ long long warp_sums[T::kThreads / 32];
    __shared__ int s_start[3];
    __shared__ uint32_t s_tmem, s_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t raw = smem_u32(smem_raw), ring = (raw + 1023u) & ~1023u;
    float *const s_merge = reinterpret_cast<float *>(smem_raw + (ring - raw) + T::kUnits * T::kUnit);
    volatile uint32_t *const abort_flag = &s_abort;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (tid == 0) {
        for (int i = 0; i < T::kUnits; ++i) {
            ncz::mbar_init(smem_u32(&bars.full[i]), kProducers);
            ncz::mbar_init(smem_u32(&bars.empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            ncz::mbar_init(smem_u32(&bars.q_full[i]), 4);
            ncz::mbar_init(smem_u32(&bars.s_full[i]), 1);
            ncz::mbar_init(smem_u32(&bars.o_done[i]), 1);
            ncz::mbar_init(smem_u32(&bars.p_full[i]), 4);
        }
        ncz::mbar_init(smem_u32(&bars.o_free), 4);
        ncz::mbar_init(smem_u32(&bars.drain[0]), 1);
        ncz::mbar_init(smem_u32(&bars.drain[1]), 1);
        s_abort = 0;
        ncz::mbar_fence_init();
    }
    if (warp == kScoreWarp) {
        ncz::tmem_alloc(smem_u32(&s_tmem), 512);
        ncz::tmem_relinquish();
    }

    // This CTA's share of the launch's tiles, as in paged_decode.
    const int unit_heads = p.by_head ? 1 : p.head_blocks;
    const int runs = p.by_head ? gridDim.x / p.head_blocks : gridDim.x;
    const int run = p.by_head ? blockIdx.x / p.head_blocks : blockIdx.x;
    const int chunk = (p.batch + T::kThreads - 1) / T::kThreads;
    const int b0 = min(tid * chunk, p.batch), b1 = min(b0 + chunk, p.batch);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) {
        int lo, hi, tiles;
        request_keys<kWideTile>(p, b, lo, hi, tiles);
        mine += static_cast<long long>(tiles) * unit_heads;
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) warp_sums[warp] = upto;
    ncz::tc_fence_before();
    __syncthreads();
    ncz::tc_fence_after();
    long long total = 0, before = upto - mine;
    for (int w = 0; w < T::kThreads / 32; ++w) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    const long long per = (total + runs - 1) / runs, first = run * per, last = min(first + per, total);
    const uint32_t tmem = s_tmem;
    if (first < last && before <= first && first < before + mine) {
        long long x = before;
        for (int b = b0; b < b1; ++b) {
            int lo, hi, tiles;
            request_keys<kWideTile>(p, b, lo, hi, tiles);
            const long long n = static_cast<long long>(tiles) * unit_heads;
            if (first < x + n) {
                s_start[0] = b;
                s_start[1] = static_cast<int>((first - x) / tiles);
                s_start[2] = static_cast<int>((first - x) % tiles);
                break;
            }
            x += n;
        }
    }
    __syncthreads();
    if (first >= last) {
        if (tid == 0 && !p.records_by_item) p.records[blockIdx.x] = make_int4(0, 0, 0, 0);
    } else {
        Cursor<kWideTile> at;
        at.b = s_start[0];
        at.hb = p.by_head ? static_cast<int>(blockIdx.x % p.head_blocks) : s_start[1];
        at.tile = s_start[2];
        request_keys<kWideTile>(p, at.b, at.lo, at.hi, at.tiles);
        const int steps = static_cast<int>(last - first);
        // Tensor memory columns: scores of two steps (128 each), O, Q of two items (D / 2 each).  Of
        // a warp's kCols scores the first half is replaced by P's high parts, the second by the low.
        const uint32_t t_o = tmem + 256, t_q = tmem + 256 + 128;

        if (warp >= kProducerWarp) {
            // ---- producers: rows 32 pw .. of every unit.
            const int pw = (warp - kProducerWarp) % kProducers, team = (warp - kProducerWarp) / kProducers;
            const int row = lane / T::kChunks, ch = lane % T::kChunks;
            const uint32_t dst0 = (ch / 8) * T::kPanel + pw * 32 * 128;
            int id = -1;
            uint32_t in_page = 0, key = 0;
            auto look_up = [&]() {
                key = static_cast<uint32_t>(at.lo & ~15) + static_cast<uint32_t>(at.tile) * kWideTile + pw * 32 + lane;
                const uint32_t col = p.page.div(key);
                in_page = key - col * p.page.d;
                id = key < static_cast<uint32_t>(at.hi) ? __ldg(p.table + at.b * p.table_stride + col) : -1;
            };
            int issued = 0, ready = 0;  // units of this warp whose copies were issued / announced
            auto unit = [&](int i) { return T::kTeams == 2 ? 2 * i + team : i; };  // K, V, K, V ..
            auto announce = [&]() {
                ncz::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars.full[unit(ready) % T::kUnits]));
                ++ready;
            };
            auto copy_unit = [&](const char *base, long long off, uint32_t mask) {
                const int slot = unit(issued) % T::kUnits, n = unit(issued) / T::kUnits;
                if (n > 0 && !__all_sync(~0u, ncz::mbar_test_wait(smem_u32(&bars.empty[slot]), (n - 1) & 1))) {
                    // Before a wait that may last: what is on its way is announced first, since the
                    // consumer may need it to get to what this warp waits for.
                    copy_wait<0>();
                    while (ready < issued) announce();
                    if (!paged_wait(&bars.empty[slot], (n - 1) & 1, abort_flag, kSiteEmpty)) return false;
                }
                const uint32_t dst = ring + slot * T::kUnit + dst0;
#pragma unroll
                for (int i = 0; i < T::kRowCopies; ++i) {
                    const int r = i * T::kRowsPerCopy + row;
                    const long long o = __shfl_sync(~0u, off, r);
                    copy16(dst + r * 128 + (((ch & 7) ^ (r & 7)) << 4), base + o + ch * 16, ((mask >> r) & 1) * 16);
                }
                copy_commit();
                ++issued;
                if (issued - ready >= T::kDepth) {
                    copy_wait<T::kDepth - 1>();
                    announce();
                }
                return true;
            };
            look_up();
            bool ok = true;
            for (int j = 0; j < steps && ok; ++j) {
                const int kv_head = p.blocks == 1 ? at.hb : at.hb / p.blocks;
                const bool in = static_cast<uint32_t>(id) < static_cast<uint32_t>(p.num_pages) &&
                                key >= static_cast<uint32_t>(at.lo);
                const uint32_t mask = __ballot_sync(~0u, in);
                // A row that is not there: zeros (0 bytes of a row that is).
                const long long k_off = in ? id * p.k_page + in_page * p.k_tok : 0;
                const long long v_off = in ? id * p.v_page + in_page * p.v_tok : 0;
                const char *const kb = p.k + kv_head * p.k_head, *const vb = p.v + kv_head * p.v_head;
                if (lane == 0 && team == 0) s_mask[j % kMaskRing][pw] = mask;  // announced with the K unit
                at.advance(p);
                if (j + 1 < steps) look_up();
                if constexpr (T::kTeams == 2)
                    ok = team == 0 ? copy_unit(kb, k_off, mask) : copy_unit(vb, v_off, mask);
                else
                    ok = copy_unit(kb, k_off, mask) && copy_unit(vb, v_off, mask);
            }
            copy_wait<0>();  // nothing of this warp is in flight when the CTA ends
            while (ready < issued) announce();
        } else if (warp == kScoreWarp) {
            // ---- Q K^T.
            constexpr uint32_t kIdescQk = ncz::umma_idesc_f16_f32(128, kWideTile, 0, 0, kBf16);
            const bool drop = g_paged_test_drop != 0 && blockIdx.x == 0;
            int item = 0;
            bool opens = true;
            for (int j = 0; j < steps; ++j) {
                const int slot = (2 * j) % T::kUnits, n = (2 * j) / T::kUnits;
                if (opens && !paged_wait(&bars.q_full[item & 1], (item >> 1) & 1, abort_flag, kSiteQFull)) break;
                if (!paged_wait(&bars.full[slot], n & 1, abort_flag, kSiteFull)) break;
                // These scores replace P of step j - 2, which P V of that step reads.
                if (j > 1 && !paged_wait(&bars.o_done[j & 1], ((j >> 1) - 1) & 1, abort_flag, kSiteODone)) break;
                ncz::tc_fence_after();
#pragma unroll
                for (int i = 0; i < T::kPanels; ++i) {
                    const uint64_t k = ncz::umma_smem_desc(ring + slot * T::kUnit + i * T::kPanel, 16, 1024, 2);
                    ncz::umma_ts_chain_elect<4>(tmem + (j & 1) * 128, t_q + (item & 1) * (D / 2) + i * 32, k, 2, kIdescQk,
                                                i > 0 ? 1u : 0u);
                }
                if (!(drop && j == 0)) ncz::umma_commit_elect(smem_u32(&bars.s_full[j & 1]));
                ncz::umma_commit_elect(smem_u32(&bars.empty[slot]));
                opens = at.tile + 1 == at.tiles;
                item += opens;
                at.advance(p);
            }
            // All MMAs are done before tensor memory is freed.
            ncz::umma_commit_elect(smem_u32(&bars.drain[0]));
            paged_wait(&bars.drain[0], 0, abort_flag, kSiteDrain, false);
        } else if (warp == kValueWarp) {
            // ---- P V.
            constexpr uint32_t kIdescPv = ncz::umma_idesc_f16_f32(128, D, 0, 1, kBf16);
            bool opens = true;
            int items = 0;  // items whose O has been taken over
            for (int j = 0; j < steps; ++j) {
                const int u = 2 * j + 1, slot = u % T::kUnits, n = u / T::kUnits;
                if (!paged_wait(&bars.full[slot], n & 1, abort_flag, kSiteFull)) break;
                if (opens && items > 0 && !paged_wait(&bars.o_free, (items - 1) & 1, abort_flag, kSiteOFree)) break;
                if (!paged_wait(&bars.p_full[j & 1], (j >> 1) & 1, abort_flag, kSiteP)) break;
                ncz::tc_fence_after();
                const uint64_t v = ncz::umma_smem_desc(ring + slot * T::kUnit, T::kPanel, 1024, 2);
                constexpr uint64_t kStep = (16 * 128) >> 4;  // 16 keys on in a V panel
                const uint32_t t_p = tmem + (j & 1) * 128, accumulate = opens ? 0u : 1u;
                if constexpr (kCopies == 1) {
                    ncz::umma_ts_chain_elect<8>(t_o, t_p, v, kStep, kIdescPv, accumulate);
                    ncz::umma_ts_chain_elect<8>(t_o, t_p + kPairs, v, kStep, kIdescPv, 1u);
                } else {
#pragma unroll
                    for (int c = 0; c < kCopies; ++c) {
                        // The lanes of copy c alone.
                        constexpr int kWords = 4 / kCopies, kSteps = kCols / 16;
                        const uint32_t at_p = t_p + c * kCols;
                        umma_ts_lanes<kSteps>(t_o, at_p, at_p + kPairs, v + c * kSteps * kStep, kStep, kIdescPv, accumulate,
                                              0 / kWords == c ? 0u : ~0u, 1 / kWords == c ? 0u : ~0u,
                                              2 / kWords == c ? 0u : ~0u, 3 / kWords == c ? 0u : ~0u);
                    }
                }
                ncz::umma_commit_elect(smem_u32(&bars.o_done[j & 1]));
                ncz::umma_commit_elect(smem_u32(&bars.empty[slot]));
                opens = at.tile + 1 == at.tiles;
                items += opens;
                at.advance(p);
            }
            ncz::umma_commit_elect(smem_u32(&bars.drain[1]));
            paged_wait(&bars.drain[1], 0, abort_flag, kSiteDrain, false);
        } else {
            // ---- softmax: query head `row` of the item, keys kCols copy .. of each step.
            const int copy = warp / (4 / kCopies), row = warp % (4 / kCopies) * 32 + lane;
            const uint32_t t_lane = static_cast<uint32_t>(warp * 32) << 16;
            const float f = fabsf(p.scale_log2);  // not 0 (paged_api.cu:choose): masked scores stay -infinity
            const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
            // Q of an item into tensor memory: this lane's query head.
            auto load_q = [&](int b, int hb, int item) {
                const int kv_head = p.blocks == 1 ? hb : hb / p.blocks;
                const int head = (hb - kv_head * p.blocks) * T::kQRows + row;
                const uint16_t *const q = reinterpret_cast<const uint16_t *>(p.q) + b * p.q_batch +
                                          (static_cast<long long>(kv_head) * p.group + head) * p.q_head;
                uint32_t w[D / 2];  // all loads first: one latency
#pragma unroll
                for (int i = 0; i < D / 2; i += 2) {
                    uint2 x = make_uint2(0, 0);
                    if (head < p.group) {
                        const uint16_t *const e = q + 2 * i;
                        if (p.q_vec)
                            x = __ldg(reinterpret_cast<const uint2 *>(e));
                        else
                            x = make_uint2(e[0] | (static_cast<uint32_t>(e[1]) << 16),
                                           e[2] | (static_cast<uint32_t>(e[3]) << 16));
                    }
                    w[i] = x.x;
                    w[i + 1] = x.y;
                }
#pragma unroll
                for (int c = 0; c < D / 2; c += 16) {
                    uint32_t x[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = w[c + i] ^ flip;
                    ncz::tmem_st_x16(t_q + t_lane + (item & 1) * (D / 2) + c, x);
                }
                ncz::tmem_wait_st();
                ncz::tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars.q_full[item & 1]));
            };
            const bool leave = g_paged_test_leave != 0 && blockIdx.x == 0 && warp == 1;
            float base = -INFINITY, sum = 0.0f;
            int item = 0;
            bool opens = true, head_cut = at.tile != 0;
            bool gave_up = false;  // this warp, at a wait; the others hear of it in softmax_together
            load_q(at.b, at.hb, 0);
            for (int j = 0; j < steps; ++j) {
                const uint32_t t_s = tmem + t_lane + (j & 1) * 128 + copy * kCols;
                gave_up = !paged_wait(&bars.s_full[j & 1], (j >> 1) & 1, abort_flag, kSiteScores);
                if (gave_up) break;
                ncz::tc_fence_after();
                uint32_t x[kCols];
                if constexpr (kCols == 32) ncz::tmem_ld_x32_wait(t_s, x);
                if constexpr (kCols == 64) ncz::tmem_ld_x64_wait(t_s, x);
                if constexpr (kCols == 128) ncz::tmem_ld_x128_wait(t_s, x);
#pragma unroll
                for (int c = 0; c < kCols / 32; ++c) {
                    const uint32_t mask = s_mask[j % kMaskRing][copy * (kCols / 32) + c];
                    if (mask != ~0u) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!((mask >> i) & 1)) x[c * 32 + i] = 0xFF800000u;
                    }
                }
                float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < kCols; ++i) t[i & 3] = fmaxf(t[i & 3], __uint_as_float(x[i]));
                const float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) * f;
                const bool grow = top > base + kTop;
                if (__any_sync(~0u, grow)) {
                    const float to = grow ? top - kLift : base;
                    const float down = base == -INFINITY ? 0.0f : grow ? ex2_approx(base - to) : 1.0f;
                    base = to;
                    sum *= down;
                    if (!opens) {
                        // O is rescaled after P V of the step before.
                        gave_up = !paged_wait(&bars.o_done[(j - 1) & 1], ((j - 1) >> 1) & 1, abort_flag, kSiteODone);
                        if (gave_up) break;
                        ncz::tc_fence_after();
#pragma unroll
                        for (int c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            ncz::tmem_ld_x16_wait(t_o + t_lane + c, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * down);
                            ncz::tmem_st_x16(t_o + t_lane + c, o);
                        }
                    }
                }
                const float m = base == -INFINITY ? 0.0f : base;
                float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < kPairs; c += 16) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int k = 2 * (c + i);
                        const float a = ex2_approx(fmaf(__uint_as_float(x[k]), f, -m));
                        const float b = ex2_approx(fmaf(__uint_as_float(x[k + 1]), f, -m));
                        s4[i & 3] += a + b;
                        hi[i] = pack16<kBf16>(a, b);
                        const float2 back = unpack16<kBf16>(hi[i]);
                        lo[i] = pack16<kBf16>(a - back.x, b - back.y);
                    }
                    ncz::tmem_st_x16(t_s + c, hi);
                    ncz::tmem_st_x16(t_s + kPairs + c, lo);
                }
                sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
                ncz::tmem_wait_st();
                ncz::tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars.p_full[j & 1]));

                if (opens) {
                    // The next item's Q, if this CTA has one: its buffer was last read before this step's scores.
                    Cursor<kWideTile> next = at;
                    next.tile = next.tiles - 1;
                    const long long left = at.tiles - at.tile;  // steps of this item
                    next.advance(p);
                    if (j + left < steps) load_q(next.b, next.hb, item + 1);
                }
                opens = false;

                const bool item_done = at.tile + 1 == at.tiles;
                if (item_done || j + 1 == steps) {
                    const bool whole = item_done && !head_cut;
                    const int kv_head = p.blocks == 1 ? at.hb : at.hb / p.blocks;
                    const int head0 = (at.hb - kv_head * p.blocks) * T::kQRows;
                    const long long part0 = static_cast<long long>(blockIdx.x * 2 + (head_cut ? 0 : 1)) * T::kQRows;
                    // Four elements of a row's O: the output, or this CTA's part of it.
                    auto put = [&](int r, int d, float4 v, float top_, float l) {
                        if (head0 + r >= p.group) return;
                        if (whole) {
                            finish_quad(p, at.b, kv_head, kv_head * p.group + head0 + r, d, v, top_, l);
                        } else {
                            *reinterpret_cast<float4 *>(p.part_o + (part0 + r) * D + d) = v;
                            if (d == 0) p.part_ml[part0 + r] = make_float2(top_, l);
                        }
                    };
                    gave_up = !paged_wait(&bars.o_done[j & 1], (j >> 1) & 1, abort_flag, kSiteODone);
                    if (leave) {
                        paged_give_up(abort_flag, kSiteMerge);
                        gave_up = true;
                    }
                    if (gave_up) break;
                    ncz::tc_fence_after();
                    if constexpr (kCopies == 1) {
#pragma unroll
                        for (int c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            ncz::tmem_ld_x16_wait(t_o + t_lane + c, o);
#pragma unroll
                            for (int i = 0; i < 16; i += 4)
                                put(row, c + i, make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]),
                                                            __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3])), base, sum);
                        }
                    } else {
                        // The copies' states through shared memory, 16 columns at a time.
                        s_ml[tid] = make_float2(base, sum);
                        if (!softmax_together(true)) break;
                        // This thread's quads of 16 columns: rows r0 + 32 i, the same ones in every chunk.
                        constexpr int kQuads = T::kQRows / 32;
                        const int r0 = tid / 4, d0 = tid % 4 * 4;
                        float to[kQuads], l[kQuads], weight[kQuads][kCopies];
#pragma unroll
                        for (int i = 0; i < kQuads; ++i) {
                            const int r = r0 + 32 * i;
                            to[i] = -INFINITY;
                            l[i] = 0.0f;
#pragma unroll
                            for (int k = 0; k < kCopies; ++k) to[i] = fmaxf(to[i], s_ml[k * T::kQRows + r].x);
#pragma unroll
                            for (int k = 0; k < kCopies; ++k) {
                                const float2 ml = s_ml[k * T::kQRows + r];
                                weight[i][k] = ml.y == 0.0f ? 0.0f : ex2_approx(ml.x - to[i]);  // 0: no keys, O is 0
                                l[i] += ml.y * weight[i][k];
                            }
                        }
#pragma unroll 2
                        for (int c = 0; c < D; c += 16) {
                            float *const buf = s_merge + (c / 16 & 1) * 128 * kMergeStride;
                            uint32_t o[16];
                            ncz::tmem_ld_x16_wait(t_o + t_lane + c, o);
#pragma unroll
                            for (int i = 0; i < 16; i += 4)
                                *reinterpret_cast<uint4 *>(buf + tid * kMergeStride + i) =
                                    make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                            softmax_sync();
#pragma unroll
                            for (int i = 0; i < kQuads; ++i) {
                                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                                for (int k = 0; k < kCopies; ++k) {
                                    const float w = weight[i][k];
                                    const float4 y = *reinterpret_cast<const float4 *>(
                                        buf + (k * T::kQRows + r0 + 32 * i) * kMergeStride + d0);
                                    v = make_float4(v.x + y.x * w, v.y + y.y * w, v.z + y.z * w, v.w + y.w * w);
                                }
                                put(r0 + 32 * i, c + d0, v, to[i], l[i]);
                            }
                        }
                        softmax_sync();  // s_ml and the last columns have been read
                    }
                    ncz::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&bars.o_free));
                    if (tid == 0) {
                        const long long end = first + j + (at.tiles - at.tile);  // first tile after the item
                        const int ctas = static_cast<int>((end - 1) / per) - run + 1;
                        const int4 rec = make_int4(at.b, at.hb, head_cut ? 0 : ctas, blockIdx.x);
                        if (p.records_by_item) {
                            if (!head_cut) p.records[static_cast<long long>(at.b) * p.head_blocks + at.hb] = rec;
                        } else if (j + 1 == steps) {
                            p.records[blockIdx.x] = rec;
                        }
                    }
                    base = -INFINITY;
                    sum = 0.0f;
                    opens = true;
                    head_cut = false;
                    ++item;
                }
                at.advance(p);
            }
            if (kCopies > 1 && gave_up) softmax_together(false);
        }
    }
    ncz::tc_fence_before();
    __syncthreads();
    ncz::tc_fence_after();
    if (warp == kScoreWarp) ncz::tmem_dealloc(tmem, 512);
}

}  // namespace nczp
