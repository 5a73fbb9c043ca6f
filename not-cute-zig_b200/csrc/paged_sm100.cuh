// paged_sm100.cuh -- the kernels of the paged key-value cache
// (include/ncz_paged.h): paged_plan, paged_append, paged_decode and
// paged_join.  Host side: paged_api.cu.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace nczp {

using ncz::ex2_approx;
using ncz::smem_u32;

// Element types of caches, inputs and outputs (the ncz_dtype numbers).
enum : int { kF32 = 0, kF16 = 1, kBF16 = 2, kE4M3 = 3 };

// Division of n < 2^31 by a fixed divisor d >= 1 as a multiply and a shift:
// with s = ceil(log2 d) and mul = floor(2^32 (2^s - d) / d) + 1,
// n / d = (n + (n * mul >> 32)) >> s  (Granlund and Montgomery, 1994).
struct FastDiv {
    uint32_t d, mul, shift;
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (n + __umulhi(n, mul)) >> shift; }
};

// A number that a generic lambda takes at compile time.
template <auto kValue>
struct Constant {
    static constexpr auto value = kValue;
};

// ---------------------------------------------------------------- plan

struct PlanParams {
    const int *held, *added, *free_pages, *free_count;
    int *table, *seq_lens;
    long long *slots;
    int *positions, *starts, *left, *status;
    long long table_stride, slot_capacity;
    int requests, width, free_capacity;
    FastDiv page;
};

constexpr int kPlanThreads = 1024;
constexpr int kPlanCluster = 8;
constexpr int kPlanRound = kPlanThreads * kPlanCluster;  // requests per round: one a thread
constexpr int kPlanSmem = kPlanRound * sizeof(int4);

__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// The address, in the cluster's window, of `addr` of CTA `rank`.
__device__ __forceinline__ uint32_t cluster_address(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_store(uint32_t addr, int x, int y) {
    asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void cluster_store(uint32_t addr, long long x, long long y) {
    asm volatile("st.shared::cluster.v2.b64 [%0], {%1, %2};" ::"r"(addr), "l"(x), "l"(y) : "memory");
}
__device__ __forceinline__ void cluster_store(uint32_t addr, const int4 &x) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w)
                 : "memory");
}

// Last i in [0, n) with start[4 i] <= x (ascending, start[0] <= x), by `bits`
// halvings of [0, 2^bits).
__device__ __forceinline__ int last_at_most(const int *start, int n, int bits, int x) {
    int r = 0;
    for (int step = bits > 0 ? 1 << (bits - 1) : 0; step > 0; step >>= 1) {
        const int at = r + step;
        if (at < n && start[4 * at] <= x) r = at;
    }
    return r;
}

// Clusters of 8 CTAs.  Per round of 8192 requests every thread of a cluster
// takes one, the CTAs scan theirs, exchange their totals, and write the prefixes
// of all requests into every CTA's shared memory.  Then each CTA writes its
// share of the round's slots and table entries, finding an entry's request by
// binary search, so that one long prompt is shared by all CTAs too.  The cluster
// barriers between reading a round's lengths and writing are what lets seq_lens
// be held, and left be free_count, in place.  Where neither is, several clusters
// do the same and share the slots and entries (PlanParams; paged_api.cu).
// Bound by latency (a few KB to 1.2 MB move): 6.4 us for 256 requests of one token, of which
// 0.9 us is an empty launch; 98304 tokens of 48 prompts 8.8 us with 16 clusters (16.2 with one);
// 8192 requests of 1 to 7 tokens 13.2 us.  0.1 us of each is the barrier that the CTAs have started.
__global__ void __cluster_dims__(kPlanCluster, 1, 1) __launch_bounds__(kPlanThreads, 1) paged_plan(const PlanParams p) {
    extern __shared__ __align__(16) char plan_smem[];
    // Of a round's requests: new tokens before it (clamped), pages asked for before it (clamped),
    // tokens held, pages held (-1 = refused).
    int4 *const s_req = reinterpret_cast<int4 *>(plan_smem);
    __shared__ long long warp_sums[32][2];
    __shared__ longlong2 s_totals[kPlanCluster];  // new tokens and pages asked for, by CTA
    __shared__ int2 s_outcome[kPlanCluster];      // pages taken up to there and requests refused, by CTA
    __shared__ int s_taken;
    // The other CTAs' shared memory may be written only once they have started: all arrive here and
    // wait in front of the first store, which the loads and the scan of round 0 lie before.
    cluster_arrive();
    const int rank = static_cast<int>(cluster_rank()), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool lead = blockIdx.x < kPlanCluster;  // the cluster that writes the lengths and counts
    const int all = blockIdx.x * kPlanThreads + tid, stride = gridDim.x * kPlanThreads;
    const int page = static_cast<int>(p.page.d);
    const long long free_count = min(max(*p.free_count, 0), p.free_capacity);
    long long tokens = 0, asked = 0;  // of the rounds before
    int taken = 0, refused = 0;       // rank 0, thread 0

    // An empty step is one round too: the barriers stand between reading free_count and writing left.
    for (int base = 0; base == 0 || base < p.requests; base += kPlanRound) {
        const int n = min(kPlanRound, p.requests - base);
        const int each = (n + kPlanCluster - 1) / kPlanCluster, bits = n > 1 ? 32 - __clz(n - 1) : 0;
        const int r = rank * each + tid;
        const bool mine = tid < each && r < n;
        const int held = mine ? p.held[base + r] : 0, added = mine ? p.added[base + r] : 0;
        const uint32_t h = max(held, 0), m = max(added, 0), end = h + m;  // < 2^32
        const int have = static_cast<int>(p.page.div(h) + (h != p.page.div(h) * p.page.d));
        const uint32_t want = end / p.page.d + (end % p.page.d != 0);
        const bool fits = held >= 0 && added >= 0 && want <= static_cast<uint32_t>(p.width);
        const int need = fits ? static_cast<int>(want) - have : 0;
        // Exclusive prefixes (a, b) over the CTA.
        long long a = m, b = need;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long xa = __shfl_up_sync(~0u, a, o), xb = __shfl_up_sync(~0u, b, o);
            if (lane >= o) {
                a += xa;
                b += xb;
            }
        }
        if (lane == 31) {
            warp_sums[warp][0] = a;
            warp_sums[warp][1] = b;
        }
        a -= m;
        b -= need;
        if (tid == 0) s_taken = 0;
        __syncthreads();
        {
            // Every warp sums the warps before it, and the CTA's total.
            long long wa = warp_sums[lane][0], wb = warp_sums[lane][1];
            long long la = lane < warp ? wa : 0, lb = lane < warp ? wb : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                wa += __shfl_xor_sync(~0u, wa, o);
                wb += __shfl_xor_sync(~0u, wb, o);
                la += __shfl_xor_sync(~0u, la, o);
                lb += __shfl_xor_sync(~0u, lb, o);
            }
            a += la;
            b += lb;
            if (base == 0) cluster_wait();  // the other CTAs have started
            if (tid < kPlanCluster) cluster_store(cluster_address(smem_u32(&s_totals[rank]), tid), wa, wb);
        }
        cluster_sync_all();  // totals; every CTA has read its lengths (and, in round 0, free_count)
        long long round_tokens = 0, round_asked = 0;
#pragma unroll
        for (int c = 0; c < kPlanCluster; ++c) {
            const longlong2 x = s_totals[c];
            if (c < rank) {
                a += x.x;
                b += x.y;
            }
            round_tokens += x.x;
            round_asked += x.y;
        }
        const bool served = fits && (need == 0 || asked + b + need <= free_count);
        const int out = __syncthreads_count(mine && !served);
        const int end_page = mine && served && need > 0 ? static_cast<int>(asked + b + need) : 0;  // <= free_count
        const int most = __reduce_max_sync(~0u, end_page);
        if (lane == 0 && most > 0) atomicMax(&s_taken, most);
        if (mine) {
            const int4 x = make_int4(static_cast<int>(min(a, 0x7FFFFFFFLL)), static_cast<int>(min(b, 0x7FFFFFFFLL)),
                                     static_cast<int>(h), served ? have : -1);
#pragma unroll
            for (int c = 0; c < kPlanCluster; ++c) cluster_store(cluster_address(smem_u32(s_req + r), c), x);
            if (lead) {
                p.seq_lens[base + r] = served ? held + added : held;
                if (p.starts != nullptr) p.starts[base + r] = static_cast<int>(min(tokens + a, p.slot_capacity));
            }
        }
        __syncthreads();  // s_taken
        if (tid == 0) cluster_store(cluster_address(smem_u32(&s_outcome[rank]), 0), s_taken, out);
        cluster_sync_all();  // the prefixes and outcomes
        if (rank == 0 && tid == 0) {
            for (int c = 0; c < kPlanCluster; ++c) {
                taken = max(taken, s_outcome[c].x);
                refused += s_outcome[c].y;
            }
        }
        // Slots and positions of the tokens.
        const int *const free_top = p.free_pages + (free_count - 1 - asked);  // read only where a page is left
        const long long room = min(round_tokens, max(0LL, p.slot_capacity - tokens));
        for (long long t = all; t < room; t += stride) {
            const int at = last_at_most(&s_req->x, n, bits, static_cast<int>(t));
            const int4 req = s_req[at];
            const uint32_t position = static_cast<uint32_t>(req.z) + static_cast<uint32_t>(static_cast<int>(t) - req.x);
            long long slot = -1;
            if (req.w >= 0) {
                const int col = static_cast<int>(p.page.div(position));
                const int id = col < req.w ? p.table[(base + at) * p.table_stride + col]
                                           : free_top[-(req.y + (col - req.w))];
                if (id >= 0) slot = static_cast<long long>(id) * page + (position - static_cast<uint32_t>(col) * page);
            }
            p.slots[tokens + t] = slot;
            if (p.positions != nullptr) p.positions[tokens + t] = static_cast<int>(min(position, 0x7FFFFFFFu));
        }
        // Table entries of the pages taken (those asked for past the stack are nobody's).
        const long long pages = min(round_asked, free_count - asked);
        for (long long i = all; i < pages; i += stride) {
            const int x = static_cast<int>(i), at = last_at_most(&s_req->y, n, bits, x);
            const int4 req = s_req[at];
            if (req.w >= 0) p.table[(base + at) * p.table_stride + req.w + (x - req.y)] = free_top[-x];
        }
        tokens += round_tokens;
        asked += round_asked;
    }
    for (long long t = tokens + all; t < p.slot_capacity; t += stride) {
        p.slots[t] = -1;
        if (p.positions != nullptr) p.positions[t] = 0;
    }
    if (lead && rank == 0 && tid == 0) {
        *p.left = static_cast<int>(free_count) - taken;
        if (p.starts != nullptr) p.starts[p.requests] = static_cast<int>(min(tokens, p.slot_capacity));
        if (p.status != nullptr) {
            p.status[0] = static_cast<int>(min(tokens, 0x7FFFFFFFLL));
            p.status[1] = taken;
            p.status[2] = refused;
            p.status[3] = static_cast<int>(min(max(0LL, tokens - p.slot_capacity), 0x7FFFFFFFLL));
        }
    }
}

// ---------------------------------------------------------------- append

struct AppendParams {
    const char *k, *v;
    char *ck, *cv;
    const float *k_scale, *v_scale;
    const long long *slots;
    long long k_tok, k_head, v_tok, v_head;                // bytes
    long long ck_page, ck_tok, ck_head, cv_page, cv_tok, cv_head;  // bytes
    long long tokens, num_slots;
    int pieces;        // pieces (kAppendPiece elements) of a token's row of one of K or V: kv_heads * head_pieces
    int head_pieces;   // head_dim / kAppendPiece
    int group;         // tokens per block
    bool vec;          // k, v and their strides are 16-byte multiples
    uint32_t page_size;
};

constexpr int kAppendThreads = 256;
constexpr int kAppendPiece = 16;  // elements of K, and as many of V, that a thread moves at once

__device__ __forceinline__ uint4 load8(const char *p, bool vec) {
    if (vec) return __ldg(reinterpret_cast<const uint4 *>(p));
    const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
    uint4 r;
    r.x = h[0] | (static_cast<uint32_t>(h[1]) << 16);
    r.y = h[2] | (static_cast<uint32_t>(h[3]) << 16);
    r.z = h[4] | (static_cast<uint32_t>(h[5]) << 16);
    r.w = h[6] | (static_cast<uint32_t>(h[7]) << 16);
    return r;
}

template <bool kBf16In>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
    if constexpr (kBf16In) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    } else {
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    }
}

// e4m3 of eight elements x / s, round to nearest even, saturating.  `below` and
// `above` are 1 / s less and more 2^-21 of it, so that x / s, rounded to f32 or
// not, lies between the two products; where both round to the same e4m3, as
// they do for all but one element in 10^5, so does it.  Only else (or where
// 1 / s leaves the normal range, below = above = 0) is the quotient computed.
// Dividing always took 10.1 us instead of 7.7 us for 10007 rows of 4 x 128 bf16.
template <int kIn>
__device__ __forceinline__ uint2 quantise8(const uint4 &x, float s, float below, float above) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t q[4], differ = below == 0.0f ? 1u : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack16<kIn == kBF16>(w[i]);
        q[i] = __nv_cvt_float2_to_fp8x2(make_float2(f.x * below, f.y * below), __NV_SATFINITE, __NV_E4M3);
        differ |= q[i] ^ __nv_cvt_float2_to_fp8x2(make_float2(f.x * above, f.y * above), __NV_SATFINITE, __NV_E4M3);
    }
    if (differ != 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack16<kIn == kBF16>(w[i]);
            q[i] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f.x, s), __fdiv_rn(f.y, s)), __NV_SATFINITE,
                                            __NV_E4M3);
        }
    }
    return make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
}

template <int kIn, bool kQuant>
__device__ __forceinline__ void append_piece(char *dst, const uint4 &x, const uint4 &y, float s) {
    if constexpr (kQuant) {
        const float inverse = 1.0f / s, size = fabsf(inverse);
        const float r = size >= 1e-37f && size <= 1e37f ? inverse : 0.0f;
        const float below = r * (1.0f - 0x1p-21f), above = r * (1.0f + 0x1p-21f);
        const uint2 a = quantise8<kIn>(x, s, below, above), b = quantise8<kIn>(y, s, below, above);
        *reinterpret_cast<uint4 *>(dst) = make_uint4(a.x, a.y, b.x, b.y);
    } else {
        reinterpret_cast<uint4 *>(dst)[0] = x;
        reinterpret_cast<uint4 *>(dst)[1] = y;
    }
}

// A thread moves 16 elements of a K row and the 16 at the same place of the V
// row: four 16-byte loads in flight.  kIn is the rows' type (read only where
// they are quantised).  Bound by HBM: 32768 rows of 8 x 64 f16, 134 MB read and
// written, 22.7 us = 5.9 TB/s; one wave of small blocks hides latency best (two or four times
// the tokens a block: 23.5 and 25.3 us).
template <int kIn, bool kQuant>
__global__ void __launch_bounds__(kAppendThreads) paged_append(const AppendParams p) {
    const long long t0 = static_cast<long long>(blockIdx.x) * p.group;
    const int count = static_cast<int>(min(static_cast<long long>(p.group), p.tokens - t0)) * p.pieces;
    for (int i = threadIdx.x; i < count; i += kAppendThreads) {
        const int local = i / p.pieces, c = i - local * p.pieces;
        const int h = c / p.head_pieces, piece = c - h * p.head_pieces;
        const long long t = t0 + local;
        const char *const k = p.k + t * p.k_tok + h * p.k_head + piece * (2 * kAppendPiece);
        const char *const v = p.v + t * p.v_tok + h * p.v_head + piece * (2 * kAppendPiece);
        const long long slot = p.slots[t];
        const uint4 k0 = load8(k, p.vec), k1 = load8(k + 16, p.vec);
        const uint4 v0 = load8(v, p.vec), v1 = load8(v + 16, p.vec);
        if (slot < 0 || slot >= p.num_slots) continue;
        const long long page = slot / p.page_size, row = slot - page * p.page_size;
        const int at = piece * kAppendPiece * (kQuant ? 1 : 2);
        const float ks = kQuant && p.k_scale != nullptr ? p.k_scale[h] : 1.0f;
        const float vs = kQuant && p.v_scale != nullptr ? p.v_scale[h] : 1.0f;
        append_piece<kIn, kQuant>(p.ck + page * p.ck_page + row * p.ck_tok + h * p.ck_head + at, k0, k1, ks);
        append_piece<kIn, kQuant>(p.cv + page * p.cv_page + row * p.cv_tok + h * p.cv_head + at, v0, v1, vs);
    }
}

// ---------------------------------------------------------------- decode

struct DecodeParams {
    const char *q, *k, *v;
    void *o;
    float *lse;
    const float *k_scale, *v_scale;
    const int *table, *lens;
    int4 *records;   // of the rows that several CTAs share: request, head block, CTAs, first CTA
    float *part_o;   // [2 * CTAs][rows][D]
    float2 *part_ml; // [2 * CTAs][rows]: maximum (log2 units) and sum
    long long k_page, k_tok, k_head, v_page, v_tok, v_head;  // bytes
    long long q_batch, q_head, o_batch, o_head, table_stride;  // elements
    int batch, group, blocks, head_blocks;  // query heads per K/V head; blocks of them; kv_heads * blocks
    int width_keys, window, num_pages;
    int whole_groups;  // page_size is a multiple of 16: the 16 keys of a group lie in one page
    int same_strides;  // K's and V's strides are equal
    int by_head;       // every CTA stays with one head block (see paged_decode)
    FastDiv page;
    float scale_log2;
    int records_by_item;
    int ctas;  // of this launch
    int q_bf16, o_dtype, q_vec, o_vec, p_parts;
};

constexpr int kWarps = 4;
constexpr int kDecodeThreads = kWarps * 32;
constexpr int kDecodeCluster = 8;  // CTAs of a cluster of paged_decode_few

// One instantiation: head_dim, cache type, and the query heads of an item, 8
// (one matrix column block, NT = 1), 16 (NT = 2) or 32 (NT = 2, two warps
// sharing each slice of keys, kShare = 2).
template <int D_, int kKv_, int kBlocks_>
struct Decode {
    static constexpr int D = D_, kKv = kKv_;
    static constexpr int NT = kBlocks_ > 1 ? 2 : 1;
    static constexpr int kShare = kBlocks_ / NT;
    static constexpr int kRows = 8 * kBlocks_;
    static constexpr int kEl = kKv == kE4M3 ? 1 : 2;
    static constexpr int kRow = D * kEl;              // bytes of a row of K or V
    static constexpr int kChunks = kRow / 16;         // 16-byte chunks of a row
    static constexpr int kRowsPerCopy = 32 / kChunks; // rows a warp's copy instruction covers
    static constexpr int kCopies = 16 / kRowsPerCopy; // copy instructions of 16 rows
    static constexpr int kSwizzles = kRowsPerCopy < 8 ? 8 / kRowsPerCopy : 1;  // different swizzles among them
    static constexpr int KS = kShare * (kRow >= 256 ? 1 : kRow >= 128 ? 2 : 4);  // 16-key groups per step
    static constexpr int kKeys = 16 * KS;                                       // keys per slice and step
    static constexpr int kSlices = kWarps / kShare;
    static constexpr int kTile = kKeys * kSlices;      // keys per CTA and step
    static constexpr int kStage = kKeys * kRow * 2;    // bytes per slice
    // CTAs per SM: as many as registers allow without spills (128, 168 or 255 a thread).  64 requests
    // of 4096 keys, 8 K/V heads, f16: head_dim 16 43.2 -> 40.2 us with four instead of three; 16
    // query heads each, head_dim 32 62.6 -> 55.8 us with three instead of two.
    static constexpr int kCtas = NT == 1 ? (kRow <= 32 ? 4 : 3) : (D <= 32 && kShare == 1 ? 3 : 2);
    static constexpr int kFit = (227 * 1024 / kCtas - 1024 - 1024) / kSlices / kStage;
    static constexpr int kStages = kFit < 6 ? kFit : 6;
    static constexpr int kSmem = kSlices * kStages * kStage;
    static constexpr int kSmemFew = kSmem + kRows * (D + 2) * 4;
    static constexpr int kMaskWords = (kKeys + 31) / 32;
    static constexpr int kCombStride = D + 4;          // floats; 4 apart: no bank conflicts when warps write
    static constexpr int MT = D / 16;                  // 16-row blocks of O^T
    static_assert(kStages >= 2 && kShare * 8 * kCombStride * 4 <= kStage, "");
};

__device__ __forceinline__ void copy16(uint32_t dst, const char *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes, or zeros where bytes is 0 (src is not read then).
__device__ __forceinline__ void copy16(uint32_t dst, const char *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
}

// Swizzle of a tile of rows of kRow bytes: the 16-byte chunk at which chunk 0
// of a row starts (xor), such that 8 rows' equal chunks lie in different banks.
template <int kRow>
__device__ __forceinline__ uint32_t chunk_xor(uint32_t row) {
    return kRow >= 128 ? row & 7 : kRow == 64 ? (row >> 1) & 3 : (row >> 2) & 1;
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// d = a b (16 x 8 x 16), starting a new sum.
template <bool kBf16>
__device__ __forceinline__ void mma16816_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    if constexpr (kBf16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    }
}
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    if constexpr (kBf16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// Two f16 of the e4m3 pair in the low half of w (exact).
__device__ __forceinline__ uint32_t e4m3_f16x2(uint32_t pair) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(pair)));
    return r;
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    return kBf16 ? ncz::pack_bf16x2(lo, hi) : ncz::pack_f16x2(lo, hi);
}

// Two elements of Q times a factor of 0: 0, or NaN where they are not finite.  With them and a factor
// of 1 a finite score is 0 and a masked one stays -infinity, which 0 times it would not.
template <bool kBf16>
__device__ __forceinline__ uint32_t times_zero16(uint32_t w) {
    constexpr uint32_t kExp = kBf16 ? 0x7F80u : 0x7C00u;  // all of it set: infinity or NaN
    const uint32_t lo = (w & kExp) == kExp ? 0x7FFFu : 0u, hi = ((w >> 16) & kExp) == kExp ? 0x7FFF0000u : 0u;
    return lo | hi;
}

// Keys of request b: [lo, hi), in `tiles` tiles from lo rounded down to 16
// (one tile at least, so that every request's rows are written).
template <int kTile>
__device__ __forceinline__ void request_keys(const DecodeParams &p, int b, int &lo, int &hi, int &tiles) {
    hi = min(max(__ldg(p.lens + b), 0), p.width_keys);
    lo = p.window > 0 ? max(0, hi - p.window) : 0;
    const uint32_t n = static_cast<uint32_t>(hi - (lo & ~15));
    tiles = max(1, static_cast<int>(n / kTile + (n % kTile != 0)));
}

// Where a CTA stands in its list of tiles: request-major, then head block
// (unless the CTA stays with one), then tile.
template <int kTile>
struct Cursor {
    int b, hb, tile, tiles, lo, hi;
    __device__ __forceinline__ void advance(const DecodeParams &p) {
        if (++tile < tiles) return;
        tile = 0;
        if (!p.by_head) {
            if (++hb < p.head_blocks) return;
            hb = 0;
        }
        if (++b < p.batch) request_keys<kTile>(p, b, lo, hi, tiles);
    }
};

__device__ __forceinline__ void store_quad(const DecodeParams &p, long long off, float4 x) {
    if (p.o_dtype == kF32) {
        float *o = static_cast<float *>(p.o) + off;
        if (p.o_vec) {
            *reinterpret_cast<float4 *>(o) = x;
        } else {
            o[0] = x.x, o[1] = x.y, o[2] = x.z, o[3] = x.w;
        }
        return;
    }
    const uint32_t lo = p.o_dtype == kBF16 ? ncz::pack_bf16x2(x.x, x.y) : ncz::pack_f16x2(x.x, x.y);
    const uint32_t hi = p.o_dtype == kBF16 ? ncz::pack_bf16x2(x.z, x.w) : ncz::pack_f16x2(x.z, x.w);
    uint16_t *o = static_cast<uint16_t *>(p.o) + off;
    if (p.o_vec) {
        *reinterpret_cast<uint2 *>(o) = make_uint2(lo, hi);
    } else {
        o[0] = lo & 0xFFFF, o[1] = lo >> 16, o[2] = hi & 0xFFFF, o[3] = hi >> 16;
    }
}

// The base of the exponentials is kept kLift below the largest score seen
// when it was set, and raised only when a score passes it by kTop: P then
// lies in (0, 2^kTop], under the largest f16 value, and keys 2^-kLift further
// down than with a base at the maximum stay above the smallest f16.  O is
// rescaled rarely (on the first keys, and where scores grow by 2^(kTop-kLift)).
constexpr float kLift = 8.0f, kTop = 15.0f;

// o = O / L * v_scale and lse = (M + log2 L) ln 2 of one query head; no keys
// (L = 0): 0 and -infinity.  M lies kLift below a score and L above 2^kLift: both are
// moved by that first, or a short row's lse were the small difference of two numbers near 8.
__device__ __forceinline__ void finish_quad(const DecodeParams &p, int b, int kv_head, int head, int d, float4 x,
                                            float m, float l) {
    const float f = l == 0.0f ? 0.0f : (p.v_scale != nullptr ? __ldg(p.v_scale + kv_head) : 1.0f) / l;
    store_quad(p, b * p.o_batch + head * p.o_head + d, make_float4(x.x * f, x.y * f, x.z * f, x.w * f));
    if (d == 0 && p.lse != nullptr) {
        const long long at = static_cast<long long>(b) * (p.head_blocks / p.blocks) * p.group + head;
        p.lse[at] = l == 0.0f ? -INFINITY : ((m + kLift) + log2f(l * 0x1p-8f)) * 0.6931471805599453f;
    }
}

__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
    float4 x;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(addr) : "memory");
    return x;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t addr) {
    float2 x;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(addr) : "memory");
    return x;
}

template <class T, bool kCluster>
__device__ __forceinline__ void decode_body(const DecodeParams &p) {
    constexpr int D = T::D, NT = T::NT, KS = T::KS, MT = T::MT, S = T::kStages;
    constexpr bool kBf16 = T::kKv == kBF16, k8 = T::kKv == kE4M3;
    extern __shared__ __align__(256) char smem[];
    __shared__ long long warp_sums[kWarps];
    __shared__ int s_start[3];
    __shared__ uint32_t s_mask[kWarps][S][T::kMaskWords];
    __shared__ float s_ml[kWarps][8][2];
    // kCluster: this CTA's part of the item, behind the ring.
    float *const s_item = reinterpret_cast<float *>(smem + T::kSmem);
    float2 *const s_item_ml = reinterpret_cast<float2 *>(s_item + T::kRows * T::D);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    const int slice = warp / T::kShare, part = warp % T::kShare;  // slice of keys, part of the query heads
    const uint32_t ring = smem_u32(smem) + slice * (S * T::kStage);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // The warps that share a slice of keys: wait for each other's copies and reads.
    auto slice_sync = [&]() {
        if constexpr (T::kShare == 1)
            __syncwarp();
        else
            asm volatile("bar.sync %0, %1;" ::"r"(1 + slice), "n"(T::kShare * 32) : "memory");
    };

    // This CTA's share of the launch's tiles: each CTA sums the requests' tile
    // counts itself (a few KB of lengths), then takes an equal run of them.
    // by_head: CTA c works on head block c % head_blocks alone, on the run
    // c / head_blocks of the tiles of all requests, so that the CTAs that read
    // one page's heads do so at the same time.
    const int unit_heads = p.by_head ? 1 : p.head_blocks;
    const int runs = p.by_head ? gridDim.x / p.head_blocks : gridDim.x;
    const int run = p.by_head ? blockIdx.x / p.head_blocks : blockIdx.x;
    long long first, last, per;
    Cursor<T::kTile> at;
    if constexpr (kCluster) {
        // One item a cluster, its tiles in eight runs.
        const int item = blockIdx.x / kDecodeCluster, rank = blockIdx.x % kDecodeCluster;
        at.b = item / p.head_blocks;
        at.hb = item % p.head_blocks;
        request_keys<T::kTile>(p, at.b, at.lo, at.hi, at.tiles);
        per = (at.tiles + kDecodeCluster - 1) / kDecodeCluster;
        first = min(rank * per, static_cast<long long>(at.tiles));
        last = min(first + per, static_cast<long long>(at.tiles));
        at.tile = static_cast<int>(first);
    } else {
        const int chunk = (p.batch + kDecodeThreads - 1) / kDecodeThreads;
        const int b0 = min(tid * chunk, p.batch), b1 = min(b0 + chunk, p.batch);
        long long mine = 0;
        for (int b = b0; b < b1; ++b) {
            int lo, hi, tiles;
            request_keys<T::kTile>(p, b, lo, hi, tiles);
            mine += static_cast<long long>(tiles) * unit_heads;
        }
        long long upto = mine;  // inclusive prefix over the warp, then exclusive over the block
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(~0u, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) warp_sums[warp] = upto;
        __syncthreads();
        long long total = 0, before = upto - mine;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += warp_sums[w];
            total += warp_sums[w];
        }
        per = (total + runs - 1) / runs;
        first = run * per;
        last = min(first + per, total);
        if (first >= last) {
            if (tid == 0 && !p.records_by_item) p.records[blockIdx.x] = make_int4(0, 0, 0, 0);
            return;
        }
        if (before <= first && first < before + mine) {
            long long x = before;
            for (int b = b0; b < b1; ++b) {
                int lo, hi, tiles;
                request_keys<T::kTile>(p, b, lo, hi, tiles);
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
        at.b = s_start[0];
        at.hb = p.by_head ? static_cast<int>(blockIdx.x % p.head_blocks) : s_start[1];
        at.tile = s_start[2];
        request_keys<T::kTile>(p, at.b, at.lo, at.hi, at.tiles);
    }

    // ---- producer side: the step being prepared is `ahead`; its keys' page
    // ids are loaded one step before its rows are copied.  A copy instruction
    // moves whole rows (kRowsPerCopy of them): lane / kChunks is its row,
    // lane % kChunks its 16-byte chunk.
    constexpr int kIds = KS > T::kMaskWords ? KS : T::kMaskWords;
    Cursor<T::kTile> ahead = at;
    long long ahead_left = last - first;
    int ids[kIds];           // page ids, -1 for keys past the end
    uint32_t in_page[kIds];  // rows in those pages
    const int row = lane / T::kChunks, chunk = lane % T::kChunks;
    const long long k_lane = row * p.k_tok + chunk * 16, v_lane = row * p.v_tok + chunk * 16;
    const long long k_copy = T::kRowsPerCopy * p.k_tok, v_copy = T::kRowsPerCopy * p.v_tok;
    uint32_t to[T::kSwizzles];  // where this lane's 16 bytes of a copy go, from the copy's first row
#pragma unroll
    for (int i = 0; i < T::kSwizzles; ++i)
        to[i] = ring + row * T::kRow + ((chunk ^ chunk_xor<T::kRow>(i * T::kRowsPerCopy + row)) << 4);
    auto first_key = [&](const Cursor<T::kTile> &c) {  // of this warp's slice, a multiple of 16
        return static_cast<uint32_t>(c.lo & ~15) + static_cast<uint32_t>(c.tile) * T::kTile + slice * T::kKeys;
    };
    auto look_up = [&]() {
        if (ahead_left <= 0) return;
        const int *const table = p.table + ahead.b * p.table_stride;
        const uint32_t key0 = first_key(ahead), hi = ahead.hi;
        if (p.whole_groups) {
            // One id per group of 16 keys, the same in every lane.
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint32_t key = key0 + i * 16, col = p.page.div(key);
                in_page[i] = key - col * p.page.d;
                ids[i] = key < hi ? __ldg(table + col) : -1;
            }
        } else {
            // Key i * 32 + lane's id.
#pragma unroll
            for (int i = 0; i < T::kMaskWords; ++i) {
                const uint32_t key = key0 + i * 32 + lane, col = p.page.div(key);
                in_page[i] = key - col * p.page.d;
                ids[i] = i * 32 + lane < T::kKeys && key < hi ? __ldg(table + col) : -1;
            }
        }
    };
    auto produce = [&](int stage) {
        if (ahead_left > 0) {
            const int kv_head = p.blocks == 1 ? ahead.hb : ahead.hb / p.blocks;
            const char *const kb = p.k + kv_head * p.k_head, *const vb = p.v + kv_head * p.v_head;
            const uint32_t key0 = first_key(ahead), lo = ahead.lo, hi = ahead.hi;
            const uint32_t at_stage = stage * T::kStage;
            constexpr uint32_t kV = T::kKeys * T::kRow;  // V's rows follow K's
            uint32_t mask[T::kMaskWords];
            if (p.whole_groups) {
#pragma unroll
                for (int i = 0; i < T::kMaskWords; ++i) mask[i] = 0;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint32_t key = key0 + ks * 16;
                    if (static_cast<uint32_t>(ids[ks]) < static_cast<uint32_t>(p.num_pages)) {  // hence key < hi
                        uint32_t m = 0xFFFFu;
                        if (hi - key < 16) m = (1u << (hi - key)) - 1;
                        if (key < lo) m &= lo - key < 16 ? ~((1u << (lo - key)) - 1) : 0u;
                        mask[ks / 2] |= m << (ks % 2 * 16);
                        const long long k_off = ids[ks] * p.k_page + in_page[ks] * p.k_tok;
                        const long long v_off = p.same_strides ? k_off : ids[ks] * p.v_page + in_page[ks] * p.v_tok;
                        const char *k_src = kb + k_off + k_lane, *v_src = vb + v_off + v_lane;
                        if (m == 0xFFFFu) {
#pragma unroll
                            for (int j = 0; j < T::kCopies; ++j) {
                                const uint32_t dst = to[j % T::kSwizzles] + at_stage +
                                                     (ks * 16 + j * T::kRowsPerCopy) * T::kRow;
                                if ((ks * T::kCopies + j) % T::kShare == part) {
                                    copy16(dst, k_src);
                                    copy16(dst + kV, v_src);
                                }
                                k_src += k_copy;
                                v_src += v_copy;
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < T::kCopies; ++j) {
                                const uint32_t dst = to[j % T::kSwizzles] + at_stage +
                                                     (ks * 16 + j * T::kRowsPerCopy) * T::kRow;
                                const uint32_t bytes = ((m >> (j * T::kRowsPerCopy + row)) & 1) * 16;
                                if ((ks * T::kCopies + j) % T::kShare == part) {
                                    copy16(dst, k_src, bytes);
                                    copy16(dst + kV, v_src, bytes);
                                }
                                k_src += k_copy;
                                v_src += v_copy;
                            }
                        }
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < T::kMaskWords; ++i) {
                    const bool ok = static_cast<uint32_t>(ids[i]) < static_cast<uint32_t>(p.num_pages) &&
                                    key0 + i * 32 + lane >= lo;
                    mask[i] = __ballot_sync(~0u, ok);
                    if (!ok) ids[i] = 0, in_page[i] = 0;  // a row of the cache, of which 0 bytes are read
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint32_t m = (mask[ks / 2] >> (ks % 2 * 16)) & 0xFFFFu;
                    if (m == 0) continue;
#pragma unroll
                    for (int j = 0; j < T::kCopies; ++j) {
                        if ((ks * T::kCopies + j) % T::kShare != part) continue;
                        const uint32_t r = j * T::kRowsPerCopy + row;
                        const int id = __shfl_sync(~0u, ids[ks / 2], (ks % 2 * 16 + r) & 31);
                        const uint32_t in = __shfl_sync(~0u, in_page[ks / 2], (ks % 2 * 16 + r) & 31);
                        const long long k_off = id * p.k_page + in * p.k_tok;
                        const long long v_off = p.same_strides ? k_off : id * p.v_page + in * p.v_tok;
                        const uint32_t dst = to[j % T::kSwizzles] + at_stage +
                                             (ks * 16 + j * T::kRowsPerCopy) * T::kRow;
                        const uint32_t bytes = ((m >> r) & 1) * 16;
                        copy16(dst, kb + k_off + chunk * 16, bytes);
                        copy16(dst + kV, vb + v_off + chunk * 16, bytes);
                    }
                }
            }
            if (lane == 0) {
#pragma unroll
                for (int i = 0; i < T::kMaskWords; ++i) s_mask[warp][stage][i] = mask[i];
            }
            ahead.advance(p);
            --ahead_left;
            look_up();
        }
        copy_commit();
    };

    look_up();
#pragma unroll 1
    for (int s = 0; s < S - 1; ++s) produce(s);

    // ---- consumer side.  Scores S^T = K Q^T (keys as rows), O^T = V^T P^T (head_dim as rows).
    float acc[MT][NT][4];  // O^T: rows g and g + 8 of block mt, query heads 2 t4 and 2 t4 + 1
    float base[NT][2], sum[NT][2];
    uint32_t qf[D / 16][NT][2];
    float f[NT][2];  // what turns a score into log2 units, above 0 (the sign is in qf)
    bool fresh = true;
    bool head_cut = at.tile != 0;  // this CTA's first item began in another CTA
    int stage = 0;
    // Rows and chunks of this lane's ldmatrix addresses: matrices 0..3 of K are
    // (keys 0-7 | 8-15) x (chunk, chunk + 1); those of V (trans) the same for e4m3 and
    // (chunk, chunk + 1) x (keys 0-7 | 8-15) for 16-bit types.
    const uint32_t k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_chunk = lane >> 4;
    const uint32_t v_row = k8 ? k_row : (lane & 7) + (lane >> 4) * 8, v_chunk = k8 ? k_chunk : (lane >> 3) & 1;
    // Address of chunk c: these ^ (c << 4) (rows and stages start on multiples of kRow).
    const uint32_t k_at = ring + k_row * T::kRow + ((k_chunk ^ chunk_xor<T::kRow>(k_row)) << 4);
    const uint32_t v_at = ring + T::kKeys * T::kRow + v_row * T::kRow + ((v_chunk ^ chunk_xor<T::kRow>(v_row)) << 4);

    for (long long step = first; step < last; ++step) {
        if (fresh) {
            fresh = false;
            const int kv_head = p.blocks == 1 ? at.hb : at.hb / p.blocks;
            const int head0 = (at.hb - kv_head * p.blocks) * T::kRows + part * (8 * NT);  // of the group
            // Over an 8-bit cache the factor has three parts whose product fits f32 where two of them may not.
            const auto scale = [&]() {
                if constexpr (k8)
                    return static_cast<double>(p.scale_log2) * (p.k_scale != nullptr ? __ldg(p.k_scale + kv_head) : 1.0f);
                else
                    return p.scale_log2;
            }();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int head = head0 + nt * 8 + g;
                const uint16_t *q = reinterpret_cast<const uint16_t *>(p.q) + at.b * p.q_batch +
                                    (static_cast<long long>(kv_head) * p.group + head) * p.q_head;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    // The elements that meet this lane's columns of the K fragments.
                    uint32_t(&w)[2] = qf[kk][nt];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int d = kk * 16 + (k8 ? 4 * t4 + 2 * j : 2 * t4 + 8 * j);
                        if (head >= p.group)
                            w[j] = 0;
                        else if (p.q_vec)
                            w[j] = __ldg(reinterpret_cast<const uint32_t *>(q + d));
                        else
                            w[j] = q[d] | (static_cast<uint32_t>(q[d + 1]) << 16);
                    }
                }
                float up = 1.0f;
                if constexpr (k8) {
                    if (p.q_bf16) {
                        // bf16 spans more than f16: take a power of two out of the row, so
                        // that its largest element lies in [1, 2); what f16 then rounds is below
                        // 2^-25 of that element.  The power is 2^-126 to 2^126, so that its inverse is a
                        // normal float too: the largest rows come to [2, 4), and rows of subnormals
                        // to multiples of 2^-7 below 1, which f16 holds exactly.
                        float top = 0.0f;
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const float2 x = unpack16<true>(qf[kk][nt][j]);
                                top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
                            }
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                        const uint32_t e = min(max((__float_as_uint(top) >> 23) & 255u, 1u), 253u);
                        up = __uint_as_float(e << 23);
                        const float down = __uint_as_float((254u - e) << 23);
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const float2 x = unpack16<true>(qf[kk][nt][j]);
                                qf[kk][nt][j] = ncz::pack_f16x2(x.x * down, x.y * down);
                            }
                    }
                }
                if (scale < 0) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                        for (int j = 0; j < 2; ++j) qf[kk][nt][j] ^= 0x80008000u;
                }
                up = static_cast<float>(up * fabs(scale));
                if (up == 0.0f) {
                    up = 1.0f;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                        for (int j = 0; j < 2; ++j) qf[kk][nt][j] = times_zero16<kBf16>(qf[kk][nt][j]);
                }
                f[nt][0] = __shfl_sync(~0u, up, (2 * t4) * 4);
                f[nt][1] = __shfl_sync(~0u, up, (2 * t4 + 1) * 4);
                base[nt][0] = base[nt][1] = -INFINITY;
                sum[nt][0] = sum[nt][1] = 0.0f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[mt][nt][e] = 0.0f;
            }
        }

        copy_wait<S - 2>();
        slice_sync();  // this stage's rows and mask are there; every lane is done with the stage before it
        produce(stage == 0 ? S - 1 : stage - 1);
        uint32_t mask[T::kMaskWords];
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < T::kMaskWords; ++i) any |= mask[i] = s_mask[warp][stage][i];
        if (any != 0) {
            const uint32_t k_src = k_at + stage * T::kStage, v_src = v_at + stage * T::kStage;
            float s[KS][NT][4];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int c = 0; c < T::kChunks; c += 2) {
                    uint32_t r[4];
                    ldmatrix4(r, (k_src ^ (c << 4)) + ks * 16 * T::kRow);
                    if constexpr (k8) {
                        // A chunk is 16 elements: two products.
                        uint32_t a[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            a[i] = e4m3_f16x2(r[i]);
                            a[4 + i] = e4m3_f16x2(r[i] >> 16);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            if (c == 0)
                                mma16816_new<false>(s[ks][nt], a[0], a[1], a[4], a[5], qf[c][nt][0], qf[c][nt][1]);
                            else
                                mma16816<false>(s[ks][nt], a[0], a[1], a[4], a[5], qf[c][nt][0], qf[c][nt][1]);
                            mma16816<false>(s[ks][nt], a[2], a[3], a[6], a[7], qf[c + 1][nt][0], qf[c + 1][nt][1]);
                        }
                    } else {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            if (c == 0)
                                mma16816_new<kBf16>(s[ks][nt], r[0], r[1], r[2], r[3], qf[0][nt][0], qf[0][nt][1]);
                            else
                                mma16816<kBf16>(s[ks][nt], r[0], r[1], r[2], r[3], qf[c / 2][nt][0], qf[c / 2][nt][1]);
                        }
                    }
                }
            }
            // Keys outside the mask: -infinity (their rows may be zeros or, where a
            // whole group is absent, an older step's).
            uint32_t every = mask[0];
#pragma unroll
            for (int i = 1; i < T::kMaskWords; ++i) every &= mask[i];
            if (every != (T::kKeys < 32 ? (1u << (T::kKeys & 31)) - 1 : ~0u)) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const bool in0 = (mask[ks / 2] >> ((ks * 16 + g) & 31)) & 1;
                    const bool in1 = (mask[ks / 2] >> ((ks * 16 + 8 + g) & 31)) & 1;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float(&x)[4] = s[ks][nt];
                        x[0] = in0 ? x[0] : -INFINITY;
                        x[1] = in0 ? x[1] : -INFINITY;
                        x[2] = in1 ? x[2] : -INFINITY;
                        x[3] = in1 ? x[3] : -INFINITY;
                    }
                }
            }
            bool grow = false;
            float top[NT][2];  // in log2 units
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const float(&x)[4] = s[ks][nt];
                    top[nt][0] = fmaxf(top[nt][0], fmaxf(x[0], x[2]));
                    top[nt][1] = fmaxf(top[nt][1], fmaxf(x[1], x[3]));
                }
                top[nt][0] *= f[nt][0];
                top[nt][1] *= f[nt][1];
                grow |= top[nt][0] > base[nt][0] + kTop || top[nt][1] > base[nt][1] + kTop;
            }
            if (__any_sync(~0u, grow)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float m = top[nt][j];
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
                        const float to = fmaxf(base[nt][j], m - kLift);
                        const float down = base[nt][j] == -INFINITY ? 0.0f : ex2_approx(base[nt][j] - to);
                        base[nt][j] = to;
                        sum[nt][j] *= down;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            acc[mt][nt][j] *= down;
                            acc[mt][nt][j + 2] *= down;
                        }
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float m0 = base[nt][0] == -INFINITY ? 0.0f : base[nt][0];
                const float m1 = base[nt][1] == -INFINITY ? 0.0f : base[nt][1];
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    float(&x)[4] = s[ks][nt];
                    x[0] = ex2_approx(fmaf(x[0], f[nt][0], -m0));
                    x[1] = ex2_approx(fmaf(x[1], f[nt][1], -m1));
                    x[2] = ex2_approx(fmaf(x[2], f[nt][0], -m0));
                    x[3] = ex2_approx(fmaf(x[3], f[nt][1], -m1));
                    sum[nt][0] += x[0] + x[2];
                    sum[nt][1] += x[1] + x[3];
                }
            }
            // P^T fragments in 16-bit parts: each takes the rounded value and leaves the rest to the next.
            uint32_t b[KS][NT][kBf16 ? 3 : 2][2];
            auto next_part = [&](int ks, int nt, int i, bool more) {
                float(&x)[4] = s[ks][nt];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t w = pack16<kBf16>(x[2 * h], x[2 * h + 1]);
                    if (more) {
                        const float2 back = unpack16<kBf16>(w);
                        x[2 * h] -= back.x;
                        x[2 * h + 1] -= back.y;
                    }
                    b[ks][nt][i][h] = transpose8x8(w);
                }
            };
            const bool two = !k8 || p.p_parts > 1;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    next_part(ks, nt, 0, two);
                    if (two) next_part(ks, nt, 1, kBf16 && p.p_parts > 2);
                    if constexpr (kBf16) {
                        if (p.p_parts > 2) next_part(ks, nt, 2, false);
                    }
                }
            // The products of a step are summed apart and then added: the
            // matrix unit's own additions cut off below 2^-24 of the sum, always downwards in
            // magnitude, which over a whole row would leave 1e-6 of it.
            auto block = [&](int ks, int nt, float (&x)[4], bool fresh_sum, uint32_t a0, uint32_t a1, uint32_t a2,
                             uint32_t a3) {
                const auto &w = b[ks][nt];
                if (fresh_sum)
                    mma16816_new<kBf16>(x, a0, a1, a2, a3, w[0][0], w[0][1]);
                else
                    mma16816<kBf16>(x, a0, a1, a2, a3, w[0][0], w[0][1]);
                if (two) mma16816<kBf16>(x, a0, a1, a2, a3, w[1][0], w[1][1]);
                if constexpr (kBf16) {
                    if (p.p_parts > 2) mma16816<kBf16>(x, a0, a1, a2, a3, w[2][0], w[2][1]);
                }
            };
            // Groups without a key are left out: their V rows are not there.
            uint32_t groups = 0;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                groups |= (((mask[ks / 2] >> (ks % 2 * 16)) & 0xFFFFu) != 0 ? 1u : 0u) << ks;
            auto products = [&](auto all_groups) {
#pragma unroll
                for (int c = 0; c < T::kChunks; c += 2) {
                    float x[k8 ? 2 : 1][NT][4];
                    if constexpr (!decltype(all_groups)::value) {
#pragma unroll
                        for (int h = 0; h < (k8 ? 2 : 1); ++h)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 4; ++e) x[h][nt][e] = 0.0f;
                    }
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        if constexpr (!decltype(all_groups)::value) {
                            if (!((groups >> ks) & 1)) continue;
                        }
                        const bool fresh_sum = decltype(all_groups)::value && ks == 0;
                        uint32_t r[4];
                        ldmatrix4_trans(r, (v_src ^ (c << 4)) + ks * 16 * T::kRow);
                        if constexpr (k8) {
                            // A register holds elements 2g, 2g + 1 of keys 2 t4, 2 t4 + 1: pair the keys.
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t lo = __byte_perm(r[2 * h], 0, 0x3120);
                                const uint32_t hi = __byte_perm(r[2 * h + 1], 0, 0x3120);
                                const uint32_t a0 = e4m3_f16x2(lo), a1 = e4m3_f16x2(lo >> 16);
                                const uint32_t a2 = e4m3_f16x2(hi), a3 = e4m3_f16x2(hi >> 16);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) block(ks, nt, x[h][nt], fresh_sum, a0, a1, a2, a3);
                            }
                        } else {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) block(ks, nt, x[0][nt], fresh_sum, r[0], r[1], r[2], r[3]);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < (k8 ? 2 : 1); ++h)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[k8 ? c + h : c / 2][nt][e] += x[h][nt][e];
                }
            };
            if (groups == (1u << KS) - 1)
                products(Constant<true>());
            else
                products(Constant<false>());
        }

        const bool item_done = at.tile + 1 == at.tiles;
        if (item_done || step + 1 == last) {
            // Join the slices' states of this item through the shared memory of the
            // stage just read, eight query heads of each part at a time.
            const bool whole = item_done && !head_cut;
            const int kv_head = p.blocks == 1 ? at.hb : at.hb / p.blocks;
            const int head0 = (at.hb - kv_head * p.blocks) * T::kRows;
            const int slot = blockIdx.x * 2 + (head_cut ? 0 : 1);
            float *const comb0 = reinterpret_cast<float *>(smem + stage * T::kStage);
            constexpr int kSliceFloats = S * T::kStage / 4;
            slice_sync();  // every lane has read the stage
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float l0 = sum[nt][0], l1 = sum[nt][1];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    l0 += __shfl_xor_sync(~0u, l0, o);
                    l1 += __shfl_xor_sync(~0u, l1, o);
                }
                if (g == 0) {
                    s_ml[warp][2 * t4][0] = base[nt][0];
                    s_ml[warp][2 * t4][1] = l0;
                    s_ml[warp][2 * t4 + 1][0] = base[nt][1];
                    s_ml[warp][2 * t4 + 1][1] = l1;
                }
                float *const out = comb0 + slice * kSliceFloats + (part * 8 + 2 * t4) * T::kCombStride;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const int d0 = mt * 16 + (k8 ? 2 * g : g), d1 = k8 ? d0 + 1 : d0 + 8;
                    out[d0] = acc[mt][nt][0];
                    out[d1] = acc[mt][nt][2];
                    out[T::kCombStride + d0] = acc[mt][nt][1];
                    out[T::kCombStride + d1] = acc[mt][nt][3];
                }
                __syncthreads();
                for (int i = tid; i < T::kShare * 8 * (D / 4); i += kDecodeThreads) {
                    const int r = i / (D / 4), d = (i % (D / 4)) * 4, of = r / 8, col = r % 8;
                    const int in_block = of * (8 * NT) + nt * 8 + col, head = head0 + in_block;
                    if (head >= p.group) continue;
                    float m = -INFINITY;
#pragma unroll
                    for (int w = 0; w < T::kSlices; ++w) m = fmaxf(m, s_ml[w * T::kShare + of][col][0]);
                    float l = 0.0f;
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < T::kSlices; ++w) {
                        const float *const ml = s_ml[w * T::kShare + of][col];
                        if (ml[1] == 0.0f) continue;  // no keys
                        const float f = ex2_approx(ml[0] - m);
                        const float4 y =
                            *reinterpret_cast<const float4 *>(comb0 + w * kSliceFloats + r * T::kCombStride + d);
                        l += ml[1] * f;
                        x = make_float4(x.x + y.x * f, x.y + y.y * f, x.z + y.z * f, x.w + y.w * f);
                    }
                    if constexpr (kCluster) {
                        *reinterpret_cast<float4 *>(s_item + in_block * D + d) = x;
                        if (d == 0) s_item_ml[in_block] = make_float2(m, l);
                    } else if (whole) {
                        finish_quad(p, at.b, kv_head, kv_head * p.group + head, d, x, m, l);
                    } else {
                        const long long to = static_cast<long long>(slot) * T::kRows + in_block;
                        *reinterpret_cast<float4 *>(p.part_o + to * D + d) = x;
                        if (d == 0) p.part_ml[to] = make_float2(m, l);
                    }
                }
                __syncthreads();
            }
            // The CTA in which an item begins says how many CTAs hold parts of it.
            if constexpr (kCluster) {
            } else if (tid == 0 && !head_cut) {
                const long long end = step + (at.tiles - at.tile);  // first tile after the item
                const int ctas = static_cast<int>((end - 1) / per) - run + 1;
                if (p.records_by_item)
                    p.records[static_cast<long long>(at.b) * p.head_blocks + at.hb] =
                        make_int4(at.b, at.hb, ctas, blockIdx.x);
                else if (step + 1 == last)
                    p.records[blockIdx.x] = make_int4(at.b, at.hb, ctas, blockIdx.x);
            } else if (tid == 0 && !p.records_by_item && step + 1 == last) {
                p.records[blockIdx.x] = make_int4(0, 0, 0, 0);  // nothing begins here and runs on
            }
            head_cut = false;
            fresh = true;
        }
        stage = stage + 1 == S ? 0 : stage + 1;
        at.advance(p);
    }

    if constexpr (kCluster) {
        // The item's eight parts, each in its CTA's shared memory, joined by all of them in
        // the same order: a share of the rows' quads each.
        if (first >= last && tid < T::kRows) s_item_ml[tid] = make_float2(-INFINITY, 0.0f);
        cluster_sync_all();
        const int item = blockIdx.x / kDecodeCluster, rank = blockIdx.x % kDecodeCluster;
        const int b = item / p.head_blocks, hb = item % p.head_blocks;
        const int kv_head = hb / p.blocks, head0 = (hb - kv_head * p.blocks) * T::kRows;
        const int quads = min(T::kRows, p.group - head0) * (D / 4);
        for (int i = rank * kDecodeThreads + tid; i < quads; i += kDecodeCluster * kDecodeThreads) {
            const int row = i / (D / 4), d = i % (D / 4) * 4;
            float2 ml[kDecodeCluster];
            float4 y[kDecodeCluster];
            float m = -INFINITY, l = 0.0f;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < kDecodeCluster; ++k) {
                ml[k] = cluster_load2(cluster_address(smem_u32(s_item_ml + row), k));
                y[k] = cluster_load4(cluster_address(smem_u32(s_item + row * D + d), k));
            }
#pragma unroll
            for (int k = 0; k < kDecodeCluster; ++k) m = fmaxf(m, ml[k].x);
#pragma unroll
            for (int k = 0; k < kDecodeCluster; ++k) {
                if (ml[k].y == 0.0f) continue;  // no keys: its O was never written
                const float w = ex2_approx(ml[k].x - m);
                l += ml[k].y * w;
                x = make_float4(x.x + y[k].x * w, x.y + y[k].y * w, x.z + y[k].z * w, x.w + y[k].w * w);
            }
            finish_quad(p, b, kv_head, kv_head * p.group + head0 + row, d, x, m, l);
        }
        cluster_sync_all();  // no CTA leaves while others read its shared memory
    }
}

// One new token per request: S^T = K Q^T, P = exp2(f S - base), O^T += V^T P^T, for the query
// heads of a K/V head at once.  4 G operations meet 2 values of K and V, so up to G = 8 to 16
// the memory bounds it: the warps are latency machines, 12 or 16 of them an SM with one stage of
// 8 KB (16 keys of 128 f16) always on its way, 96 KB an SM.  Keys are the rows of the MMAs
// (m16n8k16) and heads its 8 columns: half the accumulators and MMAs of heads as padded rows of 16,
// and a key's row is what a warp copies.  Measured: 64 requests of up to 8192 keys, 32 heads of 8,
// head_dim 128, bf16: 155 us, 6.6 TB/s; 16 heads of head_dim 64, 403 MB: 70 us, 6.4 TB/s behind
// 7.5 us of latency (launch, lengths, page ids, first rows, join).
template <class T>
__global__ void __launch_bounds__(kDecodeThreads, T::kCtas) paged_decode(const DecodeParams p) {
    decode_body<T, false>(p);
}

// The same for a few short rows: a cluster of eight CTAs per request and head block, which needs
// neither the other requests' lengths, nor a workspace, nor paged_join.  All latency: one request
// of 1000 keys, 8 K/V heads, head_dim 128, bf16: 6.9 us instead of 8.4.
template <class T>
__global__ void __cluster_dims__(kDecodeCluster, 1, 1) __launch_bounds__(kDecodeThreads, T::kCtas)
    paged_decode_few(const DecodeParams p) {
    decode_body<T, true>(p);
}

constexpr int kJoinThreads = 256;

// Joins the parts of a row.  A thread takes four elements of one query head
// (a quad) over every kJoinThreads / quads-th part; block i works on quads
// [i % per_record * quads, ...) of record i / per_record.  Few records take few
// quads per block, so that many threads share the parts of each; many take up
// to a whole item's rows, so that the grid stays within one wave of blocks.
// About 3 us behind the decode kernel (with a block per row and its parts in turn: 3 to 10).
template <int D>
__global__ void __launch_bounds__(kJoinThreads)
    paged_join(const DecodeParams p, int rows, int quads, int per_record) {
    __shared__ float4 s_o[kJoinThreads / 32][32];
    __shared__ float2 s_ml[kJoinThreads / 32][32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 rec = p.records[blockIdx.x / per_record];
    const int n = rec.z, next_cta = p.by_head ? p.head_blocks : 1;
    if (n <= 1) return;
    // A decode kernel that stopped at its wait limit leaves records unwritten: what the workspace
    // held instead is followed only where it names parts and rows of this launch.
    if (static_cast<uint32_t>(rec.x) >= static_cast<uint32_t>(p.batch) ||
        static_cast<uint32_t>(rec.y) >= static_cast<uint32_t>(p.head_blocks) || rec.w < 0 ||
        rec.w + static_cast<long long>(n - 1) * next_cta >= p.ctas)
        return;
    const int tid = threadIdx.x, lane = tid & 31;
    const int sub = tid / quads, subs = kJoinThreads / quads;
    const int quad = (blockIdx.x % per_record) * quads + tid % quads;
    const int row = quad / (D / 4), d = quad % (D / 4) * 4;
    const int kv_head = rec.y / p.blocks, head = (rec.y - kv_head * p.blocks) * rows + row;
    const bool live = row < rows && head < p.group;
    float m = -INFINITY, l = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // (m, l, x) += (m2, l2, y), both relative to their own maximum; l = 0: no keys.
    auto add = [&](float m2, float l2, float4 y) {
        const float to = fmaxf(m, m2);
        const float a = l == 0.0f ? 0.0f : ex2_approx(m - to), b = l2 == 0.0f ? 0.0f : ex2_approx(m2 - to);
        m = to;
        l = l * a + l2 * b;
        x = make_float4(x.x * a + y.x * b, x.y * a + y.y * b, x.z * a + y.z * b, x.w * a + y.w * b);
    };
    if (live) {
#pragma unroll 4
        for (int i = sub; i < n; i += subs) {
            // Part 0 is the first CTA's second slot, the others are their CTA's first.
            const long long at = static_cast<long long>((rec.w + i * next_cta) * 2 + (i == 0 ? 1 : 0)) * rows + row;
            const float2 ml = p.part_ml[at];
            add(ml.x, ml.y, *reinterpret_cast<const float4 *>(p.part_o + at * D + d));
        }
    }
    // Threads of one quad: first within the warp, then across warps.
    for (int o = quads; o < 32; o <<= 1) {
        const float m2 = __shfl_xor_sync(~0u, m, o), l2 = __shfl_xor_sync(~0u, l, o);
        const float4 y = make_float4(__shfl_xor_sync(~0u, x.x, o), __shfl_xor_sync(~0u, x.y, o),
                                     __shfl_xor_sync(~0u, x.z, o), __shfl_xor_sync(~0u, x.w, o));
        add(m2, l2, y);
    }
    if (subs > 1) {
        s_o[tid >> 5][lane] = x;
        s_ml[tid >> 5][lane] = make_float2(m, l);
        __syncthreads();
        if (tid >= quads) return;
        // With quads >= 32 a warp holds one part's share of 32 quads: the next share is quads / 32 warps on.
        const int stride = quads < 32 ? 1 : quads / 32;
        for (int w = (tid >> 5) + stride; w < kJoinThreads / 32; w += stride)
            add(s_ml[w][lane].x, s_ml[w][lane].y, s_o[w][lane]);
    }
    if (live) finish_quad(p, rec.x, kv_head, kv_head * p.group + head, d, x, m, l);
}

}  // namespace nczp
