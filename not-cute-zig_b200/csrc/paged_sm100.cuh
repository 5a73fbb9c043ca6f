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
constexpr int kPlanPer = 4;                                // requests a thread scans per round
constexpr int kPlanRound = kPlanThreads * kPlanPer;        // requests per round
constexpr int kPlanSmem = kPlanRound * 4 * sizeof(int);    // start, first page, held, flags

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// Exclusive prefix of (a, b) over the block's threads, and the block totals.
__device__ __forceinline__ void block_scan2(long long &a, long long &b, long long &total_a, long long &total_b,
                                            long long (*warp_sums)[2]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const long long own_a = a, own_b = b;
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
    __syncthreads();
    if (warp == 0) {
        long long wa = lane < warps ? warp_sums[lane][0] : 0, wb = lane < warps ? warp_sums[lane][1] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long xa = __shfl_up_sync(~0u, wa, o), xb = __shfl_up_sync(~0u, wb, o);
            if (lane >= o) {
                wa += xa;
                wb += xb;
            }
        }
        if (lane < warps) {
            warp_sums[lane][0] = wa;
            warp_sums[lane][1] = wb;
        }
    }
    __syncthreads();
    total_a = warp_sums[warps - 1][0];
    total_b = warp_sums[warps - 1][1];
    a += (warp > 0 ? warp_sums[warp - 1][0] : 0) - own_a;
    b += (warp > 0 ? warp_sums[warp - 1][1] : 0) - own_b;
    __syncthreads();
}

// Last i in [0, n) with start[i] <= x (start is ascending, start[0] <= x).
__device__ __forceinline__ int last_at_most(const int *start, int n, int x) {
    int lo = 0, hi = n;  // start[lo] <= x; hi == n or start[hi] > x
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// One cluster of 8 CTAs.  Per round of 4096 requests every CTA scans all of
// them itself (32 KB of lengths from L2, no exchange between CTAs), keeps
// the round's prefixes in shared memory, and then writes its share of the
// slots and table entries, finding each one's request by binary search.  The
// cluster barrier between reading a round's lengths and writing is what lets
// seq_lens be held, and left be free_count, in place.
__global__ void __cluster_dims__(kPlanCluster, 1, 1) __launch_bounds__(kPlanThreads, 1) paged_plan(const PlanParams p) {
    extern __shared__ int plan_smem[];
    int *const s_start = plan_smem;              // new tokens before the request, within the round (clamped)
    int *const s_first = plan_smem + kPlanRound; // pages asked for before it, within the round (clamped)
    int *const s_held = plan_smem + 2 * kPlanRound;
    int *const s_have = plan_smem + 3 * kPlanRound;  // pages held; -1 = refused
    __shared__ long long warp_sums[32][2];
    const int rank = static_cast<int>(cluster_rank()), tid = threadIdx.x;
    const int all = rank * kPlanThreads + tid, stride = kPlanCluster * kPlanThreads;
    const int page = static_cast<int>(p.page.d);
    const long long free_count = min(max(*p.free_count, 0), p.free_capacity);
    long long tokens = 0, asked = 0;  // of the rounds before
    long long taken = 0;              // this thread's largest end of a served request's pages
    int refused = 0;

    for (int base = 0; base < p.requests; base += kPlanRound) {
        const int n = min(kPlanRound, p.requests - base);
        int held[kPlanPer], added[kPlanPer], have[kPlanPer], need[kPlanPer];
        bool fits[kPlanPer];
        long long a = 0, b = 0;
#pragma unroll
        for (int i = 0; i < kPlanPer; ++i) {
            const int r = tid * kPlanPer + i;
            held[i] = r < n ? p.held[base + r] : 0;
            added[i] = r < n ? p.added[base + r] : 0;
            const uint32_t h = max(held[i], 0), m = max(added[i], 0);
            have[i] = static_cast<int>(p.page.div(h) + (h % p.page.d != 0));
            const uint32_t last = h + m;  // < 2^32
            const uint32_t want = last / p.page.d + (last % p.page.d != 0);
            fits[i] = held[i] >= 0 && added[i] >= 0 && want <= static_cast<uint32_t>(p.width);
            need[i] = fits[i] ? static_cast<int>(want) - have[i] : 0;
            a += m;
            b += need[i];
        }
        long long round_tokens, round_asked;
        block_scan2(a, b, round_tokens, round_asked, warp_sums);
        cluster_sync_all();  // every CTA has read this round's lengths (and, in round 0, free_count)
#pragma unroll
        for (int i = 0; i < kPlanPer; ++i) {
            const int r = tid * kPlanPer + i;
            if (r < n) {
                const bool served = fits[i] && (need[i] == 0 || asked + b + need[i] <= free_count);
                s_start[r] = static_cast<int>(min(a, 0x7FFFFFFFLL));
                s_first[r] = static_cast<int>(min(b, 0x7FFFFFFFLL));
                s_held[r] = max(held[i], 0);
                s_have[r] = served ? have[i] : -1;
                if (served && need[i] > 0) taken = max(taken, asked + b + need[i]);
                refused += !served;
                if (rank == r % kPlanCluster) {
                    p.seq_lens[base + r] = served ? held[i] + added[i] : held[i];
                    if (p.starts != nullptr)
                        p.starts[base + r] = static_cast<int>(min(tokens + a, p.slot_capacity));
                }
                a += max(added[i], 0);
                b += need[i];
            }
        }
        __syncthreads();
        // Slots and positions of this round's tokens.
        const long long room = min(round_tokens, max(0LL, p.slot_capacity - tokens));
        for (long long t = all; t < room; t += stride) {
            const int r = last_at_most(s_start, n, static_cast<int>(t));
            const uint32_t position = static_cast<uint32_t>(s_held[r]) + static_cast<uint32_t>(t - s_start[r]);
            const int have_r = s_have[r];
            long long slot = -1;
            if (have_r >= 0) {
                const int col = static_cast<int>(p.page.div(position));
                const int id = col < have_r
                                   ? p.table[(base + r) * p.table_stride + col]
                                   : p.free_pages[free_count - 1 - (asked + s_first[r] + (col - have_r))];
                if (id >= 0) slot = static_cast<long long>(id) * page + (position - static_cast<uint32_t>(col) * page);
            }
            p.slots[tokens + t] = slot;
            if (p.positions != nullptr) p.positions[tokens + t] = static_cast<int>(min(position, 0x7FFFFFFFu));
        }
        // Table entries of the pages taken (those asked for past the stack are nobody's).
        const long long pages = min(round_asked, free_count - asked);
        for (long long i = all; i < pages; i += stride) {
            const int r = last_at_most(s_first, n, static_cast<int>(i));
            if (s_have[r] >= 0)
                p.table[(base + r) * p.table_stride + s_have[r] + (static_cast<int>(i) - s_first[r])] =
                    p.free_pages[free_count - 1 - (asked + i)];
        }
        tokens += round_tokens;
        asked += round_asked;
        __syncthreads();
    }
    if (p.requests == 0) cluster_sync_all();  // free_count read by all before left is written
    for (long long t = tokens + all; t < p.slot_capacity; t += stride) {
        p.slots[t] = -1;
        if (p.positions != nullptr) p.positions[t] = 0;
    }
    if (rank == 0) {
        long long most = taken, sum = refused;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            most = max(most, __shfl_xor_sync(~0u, most, o));
            sum += __shfl_xor_sync(~0u, sum, o);
        }
        if ((tid & 31) == 0) {
            warp_sums[tid >> 5][0] = most;
            warp_sums[tid >> 5][1] = sum;
        }
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kPlanThreads / 32; ++w) {
                most = max(most, warp_sums[w][0]);
                sum += warp_sums[w][1];
            }
            *p.left = static_cast<int>(free_count - most);
            if (p.starts != nullptr) p.starts[p.requests] = static_cast<int>(min(tokens, p.slot_capacity));
            if (p.status != nullptr) {
                p.status[0] = static_cast<int>(min(tokens, 0x7FFFFFFFLL));
                p.status[1] = static_cast<int>(most);
                p.status[2] = static_cast<int>(sum);
                p.status[3] = static_cast<int>(min(max(0LL, tokens - p.slot_capacity), 0x7FFFFFFFLL));
            }
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
    int chunks;        // 8-element pieces of a token's row of one of K or V: kv_heads * head_dim / 8
    int head_chunks;   // head_dim / 8
    int group;         // tokens per block
    bool vec;          // k, v and their strides are 16-byte multiples
    uint32_t page_size;
};

constexpr int kAppendThreads = 256;

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

// Two e4m3 values of (a / s, b / s), round to nearest even, saturating.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b, float s) {
    const float2 x = make_float2(__fdiv_rn(a, s), __fdiv_rn(b, s));
    return __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3);
}

template <int kIn, bool kQuant>
__device__ __forceinline__ void append_piece(char *dst, const uint4 &x, float s) {
    if constexpr (kQuant) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack16<kIn == kBF16>(w[i]);
            q[i] = e4m3x2(f.x, f.y, s);
        }
        *reinterpret_cast<uint2 *>(dst) = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
    } else {
        *reinterpret_cast<uint4 *>(dst) = x;
    }
}

// A thread moves 8 elements of a K row and the 8 at the same place of the V
// row.  kIn is the rows' type (read only where they are quantised).
template <int kIn, bool kQuant>
__global__ void __launch_bounds__(kAppendThreads) paged_append(const AppendParams p) {
    const long long t0 = static_cast<long long>(blockIdx.x) * p.group;
    const int count = static_cast<int>(min(static_cast<long long>(p.group), p.tokens - t0)) * p.chunks;
    for (int i = threadIdx.x; i < count; i += kAppendThreads) {
        const int local = i / p.chunks, c = i - local * p.chunks;
        const int h = c / p.head_chunks, piece = c - h * p.head_chunks;
        const long long t = t0 + local, slot = p.slots[t];
        if (slot < 0 || slot >= p.num_slots) continue;
        const uint4 k = load8(p.k + t * p.k_tok + h * p.k_head + piece * 16, p.vec);
        const uint4 v = load8(p.v + t * p.v_tok + h * p.v_head + piece * 16, p.vec);
        const long long page = slot / p.page_size, row = slot - page * p.page_size;
        const int bytes = kQuant ? 8 : 16;
        const float ks = kQuant && p.k_scale != nullptr ? p.k_scale[h] : 1.0f;
        const float vs = kQuant && p.v_scale != nullptr ? p.v_scale[h] : 1.0f;
        append_piece<kIn, kQuant>(p.ck + page * p.ck_page + row * p.ck_tok + h * p.ck_head + piece * bytes, k, ks);
        append_piece<kIn, kQuant>(p.cv + page * p.cv_page + row * p.cv_tok + h * p.cv_head + piece * bytes, v, vs);
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
    int width_keys, window, num_pages, page_size;
    FastDiv page;
    float scale_log2;
    int min_tiles, records_by_item;
    int q_bf16, o_dtype, q_vec, o_vec, p_parts;
};

constexpr int kWarps = 4;
constexpr int kDecodeThreads = kWarps * 32;
constexpr int kCtasPerSm = 2;
constexpr int kMaxKeys = 0x7FFFFFFF;

// Copies of one 16-key group: a lane takes kKChunk bytes of the K rows g and
// g + 8 (g = lane / 4; four lanes side by side cover a row) and kVChunk bytes
// of the V rows 2t, 2t + 1, 2t + 8, 2t + 9 (t = lane % 4; eight lanes cover a
// row).  Those are exactly the rows of that lane's matrix fragments, so a
// lane reads back only bytes it copied itself and the ring needs no barrier.
template <int D_, int kKv_, int NT_>
struct Decode {
    static constexpr int D = D_, kKv = kKv_, NT = NT_;
    static constexpr int kEl = kKv == kE4M3 ? 1 : 2;
    static constexpr int kRow = D * kEl;
    static constexpr int kKChunk = kRow / 4 < 16 ? kRow / 4 : 16;
    static constexpr int kKChunks = kRow / (4 * kKChunk);
    static constexpr int kVChunk = kRow / 8 < 16 ? kRow / 8 : 16;
    static constexpr int kVChunks = kRow / (8 * kVChunk);
    static constexpr int KS = kRow >= 256 ? 1 : (kRow >= 64 ? 2 : 4);  // 16-key groups per step
    static constexpr int kKeys = 16 * KS;                              // keys per warp and step
    static constexpr int kTile = kKeys * kWarps;                       // keys per CTA and step
    static constexpr int kStage = kKeys * kRow * 2;                    // bytes per warp
    static constexpr int kStages = 24576 / kStage < 6 ? 24576 / kStage : 6;
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kMaskWords = (kKeys + 31) / 32;
    static constexpr int kRows = 8 * NT;    // query heads of an item
    static constexpr int kCombStride = D + 4;
    static constexpr bool kQSmem = D * NT > 256;  // Q fragments in shared memory where registers do not hold them
    static constexpr int kQBytes = kQSmem ? (D / 16) * NT * 32 * 8 : 0;
    static constexpr int kComb = kWarps * 8 * kCombStride * 4;
    static constexpr int kSmem = kRing + kComb + kQBytes;
    static constexpr int MT = D / 16;       // 16-row blocks of O^T
    static constexpr int CE = kKChunk / kEl, VE = kVChunk / kEl;
};

template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const char *src, uint32_t bytes) {
    if constexpr (kBytes == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    } else if constexpr (kBytes == 8) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
    }
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
}

template <int kBytes>
__device__ __forceinline__ void load_chunk(uint32_t (&r)[kBytes / 4], uint32_t addr) {
    if constexpr (kBytes == 16) {
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    } else if constexpr (kBytes == 8) {
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
    } else {
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[0]) : "r"(addr) : "memory");
    }
}

template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    if constexpr (kBf16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// Two f16 of the e4m3 pair in the low or high half of w (exact).
__device__ __forceinline__ uint32_t e4m3_f16x2(uint32_t pair) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(pair)));
    return r;
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    return kBf16 ? ncz::pack_bf16x2(lo, hi) : ncz::pack_f16x2(lo, hi);
}

// Keys of request b: [lo, hi), in `tiles` tiles (one at least, so that every
// request's rows are written).
template <int kTile>
__device__ __forceinline__ void request_keys(const DecodeParams &p, int b, int &lo, int &hi, int &tiles) {
    hi = min(max(__ldg(p.lens + b), 0), p.width_keys);
    lo = p.window > 0 ? max(0, hi - p.window) : 0;
    tiles = max(1, (hi - lo) / kTile + ((hi - lo) % kTile != 0));
}

// Where a CTA stands in the launch's list of tiles: request-major, then K/V
// head, then block of query heads, then tile.
template <int kTile>
struct Cursor {
    int b, hb, tile, tiles, lo, hi;
    __device__ __forceinline__ void advance(const DecodeParams &p) {
        if (++tile < tiles) return;
        tile = 0;
        if (++hb < p.head_blocks) return;
        hb = 0;
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

// o = O / L * v_scale and lse = (M + log2 L) ln 2 of one query head; no keys
// (L = 0): 0 and -infinity.
__device__ __forceinline__ void finish_quad(const DecodeParams &p, int b, int kv_head, int head, int d, float4 x,
                                            float m, float l) {
    const float f = l == 0.0f ? 0.0f : (p.v_scale != nullptr ? __ldg(p.v_scale + kv_head) : 1.0f) / l;
    store_quad(p, b * p.o_batch + head * p.o_head + d, make_float4(x.x * f, x.y * f, x.z * f, x.w * f));
    if (d == 0 && p.lse != nullptr) {
        const long long at = static_cast<long long>(b) * (p.head_blocks / p.blocks) * p.group + head;
        p.lse[at] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
}

// The base of the exponentials is kept kLift below the largest score seen
// when it was set, and raised only when a score passes it by kTop: P then
// lies in (0, 2^kTop], under the largest f16 value, keys 2^-kLift of the
// f16 range's bottom above what a base at the maximum would keep, and O is
// rescaled rarely (on the first keys, and where scores grow by 2^(kTop-kLift)).
constexpr float kLift = 8.0f, kTop = 15.0f;

template <class T>
__global__ void __launch_bounds__(kDecodeThreads, T::kSmem > 113 * 1024 ? 1 : kCtasPerSm)
    paged_decode(const DecodeParams p) {
    constexpr int D = T::D, NT = T::NT, KS = T::KS, MT = T::MT, S = T::kStages;
    constexpr bool kBf16 = T::kKv == kBF16, k8 = T::kKv == kE4M3;
    extern __shared__ __align__(16) char smem[];
    __shared__ long long warp_sums[kWarps];
    __shared__ int s_start[3];
    __shared__ uint32_t s_mask[kWarps][S][T::kMaskWords];
    __shared__ float s_ml[kWarps][8][2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    float *const comb = reinterpret_cast<float *>(smem + T::kRing);
    const uint32_t ring = smem_u32(smem) + warp * (S * T::kStage);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // This CTA's share of the launch's tiles: each CTA sums the requests' tile
    // counts itself (a few KB of lengths), then takes an equal run of tiles.
    long long first, last;  // [first, last)
    long long per;
    Cursor<T::kTile> at;
    {
        const int chunk = (p.batch + kDecodeThreads - 1) / kDecodeThreads;
        const int b0 = min(tid * chunk, p.batch), b1 = min(b0 + chunk, p.batch);
        long long mine = 0;
        for (int b = b0; b < b1; ++b) {
            int lo, hi, tiles;
            request_keys<T::kTile>(p, b, lo, hi, tiles);
            mine += static_cast<long long>(tiles) * p.head_blocks;
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
        per = max((total + gridDim.x - 1) / gridDim.x, static_cast<long long>(p.min_tiles));
        first = blockIdx.x * per;
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
                const long long n = static_cast<long long>(tiles) * p.head_blocks;
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
        at.hb = s_start[1];
        at.tile = s_start[2];
        request_keys<T::kTile>(p, at.b, at.lo, at.hi, at.tiles);
    }

    // ---- producer side: the step being prepared is `ahead`; its keys' page
    // ids are loaded one step before its rows are copied.
    constexpr int kOwn = T::kMaskWords;  // keys a lane looks up per step
    Cursor<T::kTile> ahead = at;
    long long ahead_left = last - first;
    int ids[kOwn];
    auto look_up = [&]() {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const long long key = static_cast<long long>(ahead.lo) + static_cast<long long>(ahead.tile) * T::kTile +
                                  warp * T::kKeys + i * 32 + lane;
            ids[i] = -1;
            if (ahead_left > 0 && i * 32 + lane < T::kKeys && key < ahead.hi)
                ids[i] = __ldg(p.table + ahead.b * p.table_stride + p.page.div(static_cast<uint32_t>(key)));
        }
    };
    auto produce = [&](int stage) {
        if (ahead_left > 0) {
            const int kv_head = p.blocks == 1 ? ahead.hb : ahead.hb / p.blocks;
            const char *const kb = p.k + kv_head * p.k_head, *const vb = p.v + kv_head * p.v_head;
            long long k_off[kOwn], v_off[kOwn];
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < kOwn; ++i) {
                const uint32_t key = static_cast<uint32_t>(ahead.lo) + static_cast<uint32_t>(ahead.tile) * T::kTile +
                                     warp * T::kKeys + i * 32 + lane;  // used only where it is below hi
                const bool ok = ids[i] >= 0 && ids[i] < p.num_pages;
                const int row = ok ? static_cast<int>(key - p.page.div(key) * p.page.d) : 0;
                k_off[i] = ok ? ids[i] * p.k_page + row * p.k_tok : -1;
                v_off[i] = ok ? ids[i] * p.v_page + row * p.v_tok : -1;
                const uint32_t mask = __ballot_sync(~0u, ok);
                any |= mask;
                if (lane == 0) s_mask[warp][stage][i] = mask;
            }
            if (any != 0) {
                const uint32_t k_dst = ring + stage * T::kStage + lane * T::kKChunk;
                const uint32_t v_dst = ring + stage * T::kStage + T::kKeys * T::kRow + lane * T::kVChunk;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const long long off = __shfl_sync(~0u, k_off[ks / 2], (ks * 16 + r * 8 + g) & 31);
                        const char *src = kb + (off >= 0 ? off + t4 * T::kKChunk : 0);
                        const uint32_t bytes = off >= 0 ? T::kKChunk : 0;
#pragma unroll
                        for (int c = 0; c < T::kKChunks; ++c)
                            copy_async<T::kKChunk>(k_dst + ((ks * 2 + r) * T::kKChunks + c) * (32 * T::kKChunk),
                                                   src + (off >= 0 ? c * 4 * T::kKChunk : 0), bytes);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const long long off =
                            __shfl_sync(~0u, v_off[ks / 2], (ks * 16 + (r >> 1) * 8 + t4 * 2 + (r & 1)) & 31);
                        const char *src = vb + (off >= 0 ? off + g * T::kVChunk : 0);
                        const uint32_t bytes = off >= 0 ? T::kVChunk : 0;
#pragma unroll
                        for (int c = 0; c < T::kVChunks; ++c)
                            copy_async<T::kVChunk>(v_dst + ((ks * 4 + r) * T::kVChunks + c) * (32 * T::kVChunk),
                                                   src + (off >= 0 ? c * 8 * T::kVChunk : 0), bytes);
                    }
                }
            }
            ahead.advance(p);
            --ahead_left;
            look_up();
        }
        copy_commit();
    };

    look_up();
#pragma unroll
    for (int s = 0; s < S - 1; ++s) produce(s);

    // ---- consumer side
    float acc[MT][NT][4];  // O^T: rows g and g + 8 of block mt, query heads 2 t4 and 2 t4 + 1
    float base[NT][2], sum[NT][2];
    uint32_t qf[T::kQSmem ? 1 : D / 16][NT][2];
    float q_up[NT][2];  // power of two taken out of a query head's elements (bf16 q against an e4m3 cache)
    uint2 *const s_q = reinterpret_cast<uint2 *>(smem + T::kRing + T::kComb);
    bool fresh = true;
    bool head_cut = at.tile != 0;  // this CTA's first item began in another CTA
    int stage = 0;
    float scale = 0.0f;
    for (long long step = first; step < last; ++step) {
        if (fresh) {
            fresh = false;
            const int kv_head = p.blocks == 1 ? at.hb : at.hb / p.blocks;
            const int head0 = (at.hb - kv_head * p.blocks) * T::kRows;  // first query head of the group
            scale = p.scale_log2 * (k8 && p.k_scale != nullptr ? __ldg(p.k_scale + kv_head) : 1.0f);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int head = head0 + nt * 8 + g;
                const uint16_t *q = reinterpret_cast<const uint16_t *>(p.q) + at.b * p.q_batch +
                                    (static_cast<long long>(kv_head) * p.group + head) * p.q_head;
                uint32_t w[D / 16][2];
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    // The elements of this lane's pieces of the K rows, in their order.
                    const int d = (kk / (T::CE / 4)) * (4 * T::CE) + t4 * T::CE + (kk % (T::CE / 4)) * 4;
                    if (head >= p.group) {
                        w[kk][0] = w[kk][1] = 0;
                    } else if (p.q_vec) {
                        const uint2 x = __ldg(reinterpret_cast<const uint2 *>(q + d));
                        w[kk][0] = x.x;
                        w[kk][1] = x.y;
                    } else {
                        w[kk][0] = q[d] | (static_cast<uint32_t>(q[d + 1]) << 16);
                        w[kk][1] = q[d + 2] | (static_cast<uint32_t>(q[d + 3]) << 16);
                    }
                }
                float up = 1.0f;
                if constexpr (k8) {
                    if (p.q_bf16) {
                        // bf16 spans more than f16: take a power of two out of the row, so
                        // that its largest element lies in [1, 2); what f16 then rounds is below
                        // 2^-25 of that element.
                        float top = 0.0f;
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const float2 f = unpack16<true>(w[kk][j]);
                                top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                            }
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                        const uint32_t e = (__float_as_uint(top) >> 23) & 255u;
                        // 2^(e-127) and its inverse, both normal floats for 1 <= e <= 253
                        const bool in = e >= 1 && e <= 253;
                        up = in ? __uint_as_float(e << 23) : 1.0f;
                        const float down = in ? __uint_as_float((254u - e) << 23) : 1.0f;
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const float2 f = unpack16<true>(w[kk][j]);
                                w[kk][j] = ncz::pack_f16x2(f.x * down, f.y * down);
                            }
                    }
                    q_up[nt][0] = __shfl_sync(~0u, up, (2 * t4) * 4);
                    q_up[nt][1] = __shfl_sync(~0u, up, (2 * t4 + 1) * 4);
                }
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    if constexpr (T::kQSmem) {
                        // All warps hold the same fragments: each writes the same bytes.
                        s_q[(kk * NT + nt) * 32 + lane] = make_uint2(w[kk][0], w[kk][1]);
                    } else {
                        qf[kk][nt][0] = w[kk][0];
                        qf[kk][nt][1] = w[kk][1];
                    }
                }
                base[nt][0] = base[nt][1] = -INFINITY;
                sum[nt][0] = sum[nt][1] = 0.0f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[mt][nt][e] = 0.0f;
            }
            if constexpr (T::kQSmem) __syncwarp();
        }

        copy_wait<S - 2>();
        __syncwarp();  // lane 0's mask words of this stage; every lane is done with the stage before it
        produce(stage == 0 ? S - 1 : stage - 1);
        uint32_t mask[T::kMaskWords];
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < T::kMaskWords; ++i) any |= mask[i] = s_mask[warp][stage][i];
        if (any != 0) {
            const uint32_t k_src = ring + stage * T::kStage + lane * T::kKChunk;
            const uint32_t v_src = ring + stage * T::kStage + T::kKeys * T::kRow + lane * T::kVChunk;
            float s[KS][NT][4];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[ks][nt][e] = 0.0f;
#pragma unroll
                for (int c = 0; c < T::kKChunks; ++c) {
                    uint32_t ra[T::kKChunk / 4], rb[T::kKChunk / 4];
                    load_chunk<T::kKChunk>(ra, k_src + ((ks * 2 + 0) * T::kKChunks + c) * (32 * T::kKChunk));
                    load_chunk<T::kKChunk>(rb, k_src + ((ks * 2 + 1) * T::kKChunks + c) * (32 * T::kKChunk));
#pragma unroll
                    for (int i = 0; i < T::CE / 4; ++i) {
                        uint32_t a0, a1, a2, a3;
                        if constexpr (k8) {
                            a0 = e4m3_f16x2(ra[i]);
                            a1 = e4m3_f16x2(rb[i]);
                            a2 = e4m3_f16x2(ra[i] >> 16);
                            a3 = e4m3_f16x2(rb[i] >> 16);
                        } else {
                            a0 = ra[2 * i];
                            a1 = rb[2 * i];
                            a2 = ra[2 * i + 1];
                            a3 = rb[2 * i + 1];
                        }
                        const int kk = c * (T::CE / 4) + i;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            uint32_t b0, b1;
                            if constexpr (T::kQSmem) {
                                const uint2 x = s_q[(kk * NT + nt) * 32 + lane];
                                b0 = x.x;
                                b1 = x.y;
                            } else {
                                b0 = qf[kk][nt][0];
                                b1 = qf[kk][nt][1];
                            }
                            mma16816<kBf16>(s[ks][nt], a0, a1, a2, a3, b0, b1);
                        }
                    }
                }
            }
            // Scores in log2 units; keys outside the mask -infinity.
            bool grow = false;
            float top[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float f0 = k8 ? scale * q_up[nt][0] : scale, f1 = k8 ? scale * q_up[nt][1] : scale;
                top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const bool in0 = (mask[ks / 2] >> ((ks * 16 + g) & 31)) & 1;
                    const bool in1 = (mask[ks / 2] >> ((ks * 16 + 8 + g) & 31)) & 1;
                    float(&x)[4] = s[ks][nt];
                    x[0] = in0 ? x[0] * f0 : -INFINITY;
                    x[1] = in0 ? x[1] * f1 : -INFINITY;
                    x[2] = in1 ? x[2] * f0 : -INFINITY;
                    x[3] = in1 ? x[3] * f1 : -INFINITY;
                    top[nt][0] = fmaxf(top[nt][0], fmaxf(x[0], x[2]));
                    top[nt][1] = fmaxf(top[nt][1], fmaxf(x[1], x[3]));
                }
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
                        const float f = base[nt][j] == -INFINITY ? 0.0f : ex2_approx(base[nt][j] - to);
                        base[nt][j] = to;
                        sum[nt][j] *= f;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            acc[mt][nt][j] *= f;
                            acc[mt][nt][j + 2] *= f;
                        }
                    }
            }
            uint32_t pb[KS][NT][2][2];  // [part][key half]: P^T fragments
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float m0 = base[nt][0] == -INFINITY ? 0.0f : base[nt][0];
                const float m1 = base[nt][1] == -INFINITY ? 0.0f : base[nt][1];
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    float(&x)[4] = s[ks][nt];
                    x[0] = ex2_approx(x[0] - m0);
                    x[1] = ex2_approx(x[1] - m1);
                    x[2] = ex2_approx(x[2] - m0);
                    x[3] = ex2_approx(x[3] - m1);
                    sum[nt][0] += x[0] + x[2];
                    sum[nt][1] += x[1] + x[3];
                }
            }
            // P in 16-bit parts: each takes the rounded value and leaves the rest to the next.
            auto next_part = [&](int ks, int nt, uint32_t (&b)[2]) {
                float(&x)[4] = s[ks][nt];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t w = pack16<kBf16>(x[2 * h], x[2 * h + 1]);
                    const float2 back = unpack16<kBf16>(w);
                    x[2 * h] -= back.x;
                    x[2 * h + 1] -= back.y;
                    b[h] = transpose8x8(w);
                }
            };
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    next_part(ks, nt, pb[ks][nt][0]);
                    next_part(ks, nt, pb[ks][nt][1]);
                }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t third[NT][2];
                if constexpr (kBf16) {
                    if (p.p_parts > 2) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) next_part(ks, nt, third[nt]);
                    }
                }
#pragma unroll
                for (int c = 0; c < T::kVChunks; ++c) {
                    uint32_t r[4][T::kVChunk / 4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        load_chunk<T::kVChunk>(r[i], v_src + ((ks * 4 + i) * T::kVChunks + c) * (32 * T::kVChunk));
#pragma unroll
                    for (int m = 0; m < T::VE / 2; ++m) {
                        // Rows of V^T: two elements of each row, keys paired.
                        uint32_t a0, a1, a2, a3;
                        if constexpr (k8) {
                            const uint32_t sel = m % 2 == 0 ? 0x5140 : 0x7362;
                            const uint32_t x = __byte_perm(r[0][m / 2], r[1][m / 2], sel);
                            const uint32_t y = __byte_perm(r[2][m / 2], r[3][m / 2], sel);
                            a0 = e4m3_f16x2(x);
                            a1 = e4m3_f16x2(x >> 16);
                            a2 = e4m3_f16x2(y);
                            a3 = e4m3_f16x2(y >> 16);
                        } else {
                            a0 = __byte_perm(r[0][m], r[1][m], 0x5410);
                            a1 = __byte_perm(r[0][m], r[1][m], 0x7632);
                            a2 = __byte_perm(r[2][m], r[3][m], 0x5410);
                            a3 = __byte_perm(r[2][m], r[3][m], 0x7632);
                        }
                        const int mt = c * (T::VE / 2) + m;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816<kBf16>(acc[mt][nt], a0, a1, a2, a3, pb[ks][nt][0][0], pb[ks][nt][0][1]);
                            mma16816<kBf16>(acc[mt][nt], a0, a1, a2, a3, pb[ks][nt][1][0], pb[ks][nt][1][1]);
                            if constexpr (kBf16) {
                                if (p.p_parts > 2)
                                    mma16816<kBf16>(acc[mt][nt], a0, a1, a2, a3, third[nt][0], third[nt][1]);
                            }
                        }
                    }
                }
            }
        }
        stage = stage + 1 == S ? 0 : stage + 1;

        const bool item_done = at.tile + 1 == at.tiles;
        if (item_done || step + 1 == last) {
            // Join the warps' states of this item through shared memory, eight query heads at a time.
            const bool whole = item_done && !head_cut;
            const int kv_head = p.blocks == 1 ? at.hb : at.hb / p.blocks;
            const int head0 = (at.hb - kv_head * p.blocks) * T::kRows;
            const int slot = blockIdx.x * 2 + (head_cut ? 0 : 1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (head0 + nt * 8 >= p.group) break;
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
                float *const out = comb + (warp * 8 + 2 * t4) * T::kCombStride;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const int d = (mt / (T::VE / 2)) * (8 * T::VE) + g * T::VE + 2 * (mt % (T::VE / 2));
                    *reinterpret_cast<float2 *>(out + d) = make_float2(acc[mt][nt][0], acc[mt][nt][2]);
                    *reinterpret_cast<float2 *>(out + T::kCombStride + d) =
                        make_float2(acc[mt][nt][1], acc[mt][nt][3]);
                }
                __syncthreads();
                for (int i = tid; i < 8 * (D / 4); i += kDecodeThreads) {
                    const int r = i / (D / 4), d = (i % (D / 4)) * 4, head = head0 + nt * 8 + r;
                    if (head >= p.group) break;
                    float m = -INFINITY;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_ml[w][r][0]);
                    float l = 0.0f;
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        if (s_ml[w][r][1] == 0.0f) continue;  // no keys
                        const float f = ex2_approx(s_ml[w][r][0] - m);
                        const float4 y = *reinterpret_cast<const float4 *>(comb + (w * 8 + r) * T::kCombStride + d);
                        l += s_ml[w][r][1] * f;
                        x = make_float4(x.x + y.x * f, x.y + y.y * f, x.z + y.z * f, x.w + y.w * f);
                    }
                    if (whole) {
                        finish_quad(p, at.b, kv_head, kv_head * p.group + head, d, x, m, l);
                    } else {
                        const long long row = static_cast<long long>(slot) * T::kRows + nt * 8 + r;
                        *reinterpret_cast<float4 *>(p.part_o + row * D + d) = x;
                        if (d == 0) p.part_ml[row] = make_float2(m, l);
                    }
                }
                __syncthreads();
            }
            // The CTA in which an item begins says how many CTAs hold parts of it.
            if (tid == 0 && !head_cut) {
                const long long end = step + (at.tiles - at.tile);  // first tile after the item
                const int ctas = static_cast<int>((end - 1) / per - blockIdx.x) + 1;
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
        at.advance(p);
    }
}

constexpr int kJoinThreads = 256;

// Joins the parts of one query head's row: block (record, row).  D / 4 threads
// take one part's row together, kJoinThreads / (D / 4) parts at a time.
template <int D>
__global__ void __launch_bounds__(kJoinThreads) paged_join(const DecodeParams p, int rows, int row_stride) {
    constexpr int kLanes = D / 4, kSubs = kJoinThreads / kLanes;
    __shared__ float s_max[kJoinThreads / 32];
    __shared__ float s_sum[kSubs];
    __shared__ float4 s_o[kSubs][kLanes];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 rec = p.records[blockIdx.x / rows];
    const int n = rec.z;
    if (n <= 1) return;
    const int row = blockIdx.x % rows;
    const int kv_head = rec.y / p.blocks, head = (rec.y - kv_head * p.blocks) * row_stride + row;
    if (head >= p.group) return;
    const int tid = threadIdx.x;
    // Part 0 is the first CTA's second slot, the others are their CTA's first.
    auto at = [&](int i) {
        return static_cast<long long>((rec.w + i) * 2 + (i == 0 ? 1 : 0)) * row_stride + row;
    };
    float m = -INFINITY;
    for (int i = tid; i < n; i += kJoinThreads) m = fmaxf(m, p.part_ml[at(i)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if ((tid & 31) == 0) s_max[tid >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) m = fmaxf(m, s_max[w]);
    const int sub = tid / kLanes, q = tid % kLanes;
    float l = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = sub; i < n; i += kSubs) {
        const float2 ml = p.part_ml[at(i)];
        const float4 y = *reinterpret_cast<const float4 *>(p.part_o + at(i) * D + q * 4);
        const float f = ml.y == 0.0f ? 0.0f : ex2_approx(ml.x - m);  // 0: no keys
        l += ml.y * f;
        x = make_float4(x.x + y.x * f, x.y + y.y * f, x.z + y.z * f, x.w + y.w * f);
    }
    s_o[sub][q] = x;
    if (q == 0) s_sum[sub] = l;
    __syncthreads();
    if (sub != 0) return;
    for (int s = 1; s < kSubs; ++s) {
        const float4 y = s_o[s][q];
        l += s_sum[s];
        x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
    }
    finish_quad(p, rec.x, kv_head, kv_head * p.group + head, q * 4, x, m, l);
}

}  // namespace nczp
