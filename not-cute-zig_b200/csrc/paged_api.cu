// paged_api.cu -- the C ABI of the paged key-value cache (include/ncz_paged.h)
// over the kernels of paged_sm100.cuh.
#include <algorithm>
#include <cstdint>
#include <cstring>
#include <mutex>

#include "driver.cuh"
#include "ncz_flash.h"
#include "ncz_paged.h"
#include "paged_wide_sm100.cuh"
#include "status.cuh"

namespace {

using ncz::drv;
using ncz::map_cuda_error;

constexpr int kMaxDevices = 64;
constexpr size_t kMaxInt = 0x7FFFFFFF;
constexpr size_t kMaxRequests = size_t(1) << 24;
constexpr size_t kMaxStride = size_t(1) << 40;  // elements; offsets then stay far inside 64 bits

constexpr size_t kPlanClusters = 16, kSlotsPerCluster = 4096;

std::mutex g_mu;
int g_sms[kMaxDevices];

// Held over a decode launch and its join, by stream: another thread's decode on the same stream,
// which may use the same workspace, must not come between the two.
std::mutex g_pair_mu[64];
std::mutex &pair_mutex(int dev, const void *stream) {
    return g_pair_mu[(reinterpret_cast<uintptr_t>(stream) / 64 * 31 + static_cast<uintptr_t>(dev)) % 64];
}

// One instantiation: its address, label, shared memory and what of it has been set up.
struct Kernel {
    const void *fn;
    const char *label;
    int smem;
    int ctas;  // decode: CTAs per SM
    int tile;  // decode: keys a CTA takes per step
    int threads;
    bool ready[kMaxDevices];
};

template <int D, int kKv, int NT>
const void *decode_fn() {
    return reinterpret_cast<const void *>(nczp::paged_decode<nczp::Decode<D, kKv, NT>>);
}
#define NCZ_DECODE(D, KV, KVNAME, NT) \
    {decode_fn<D, KV, NT>(), "paged_decode<" #D "," KVNAME "," #NT ">", nczp::Decode<D, KV, NT>::kSmem, \
     nczp::Decode<D, KV, NT>::kCtas, nczp::Decode<D, KV, NT>::kTile, nczp::kDecodeThreads, {}}
template <int D, int kKv, int NT>
const void *few_fn() {
    return reinterpret_cast<const void *>(nczp::paged_decode_few<nczp::Decode<D, kKv, NT>>);
}
#define NCZ_FEW(D, KV, KVNAME, NT) \
    {few_fn<D, KV, NT>(), "paged_decode_few<" #D "," KVNAME "," #NT ">", nczp::Decode<D, KV, NT>::kSmemFew, \
     nczp::Decode<D, KV, NT>::kCtas, nczp::Decode<D, KV, NT>::kTile, nczp::kDecodeThreads, {}}
#define NCZ_FEW_NT(D, KV, KVNAME) {NCZ_FEW(D, KV, KVNAME, 1), NCZ_FEW(D, KV, KVNAME, 2)}
#define NCZ_FEW_D(KV, KVNAME, FIRST) \
    {FIRST, NCZ_FEW_NT(32, KV, KVNAME), NCZ_FEW_NT(64, KV, KVNAME), NCZ_FEW_NT(128, KV, KVNAME)}

#define NCZ_DECODE_NT(D, KV, KVNAME) \
    {NCZ_DECODE(D, KV, KVNAME, 1), NCZ_DECODE(D, KV, KVNAME, 2), NCZ_DECODE(D, KV, KVNAME, 4)}
#define NCZ_DECODE_D(KV, KVNAME, FIRST) \
    {FIRST, NCZ_DECODE_NT(32, KV, KVNAME), NCZ_DECODE_NT(64, KV, KVNAME), NCZ_DECODE_NT(128, KV, KVNAME)}
#define NCZ_NONE {{nullptr, nullptr, 0, 0, 0, 0, {}}, {nullptr, nullptr, 0, 0, 0, 0, {}}, {nullptr, nullptr, 0, 0, 0, 0, {}}}

// [cache type - 1][log2(head_dim) - 4][log2(query heads per item / 8)]
Kernel g_decode[3][4][3] = {
    NCZ_DECODE_D(nczp::kF16, "f16", NCZ_DECODE_NT(16, nczp::kF16, "f16")),
    NCZ_DECODE_D(nczp::kBF16, "bf16", NCZ_DECODE_NT(16, nczp::kBF16, "bf16")),
    NCZ_DECODE_D(nczp::kE4M3, "e4m3", NCZ_NONE),
};
// The same for clusters, up to 16 query heads an item.
Kernel g_few[3][4][2] = {
    NCZ_FEW_D(nczp::kF16, "f16", NCZ_FEW_NT(16, nczp::kF16, "f16")),
    NCZ_FEW_D(nczp::kBF16, "bf16", NCZ_FEW_NT(16, nczp::kBF16, "bf16")),
    {{{nullptr, nullptr, 0, 0, 0, 0, {}}, {nullptr, nullptr, 0, 0, 0, 0, {}}},
     NCZ_FEW_NT(32, nczp::kE4M3, "e4m3"), NCZ_FEW_NT(64, nczp::kE4M3, "e4m3"), NCZ_FEW_NT(128, nczp::kE4M3, "e4m3")},
};
template <int D, bool kBf16, int kQRows>
const void *wide_fn() {
    return reinterpret_cast<const void *>(nczp::paged_decode_wide<nczp::Wide<D, kBf16, kQRows>>);
}
#define NCZ_WIDE(D, BF16, NAME, ROWS) \
    {wide_fn<D, BF16, ROWS>(), "paged_decode_wide<" #D "," NAME "," #ROWS ">", nczp::Wide<D, BF16, ROWS>::kSmem, 1, \
     nczp::kWideTile, nczp::Wide<D, BF16, ROWS>::kThreads, {}}

#define NCZ_WIDE_ROWS(D, BF16, NAME) \
    {NCZ_WIDE(D, BF16, NAME, 32), NCZ_WIDE(D, BF16, NAME, 64), NCZ_WIDE(D, BF16, NAME, 128)}

// [bf16][head_dim 64, 128][32, 64, 128 query heads]
Kernel g_wide[2][2][3] = {
    {NCZ_WIDE_ROWS(64, false, "f16"), NCZ_WIDE_ROWS(128, false, "f16")},
    {NCZ_WIDE_ROWS(64, true, "bf16"), NCZ_WIDE_ROWS(128, true, "bf16")},
};
Kernel g_join[4] = {
    {reinterpret_cast<const void *>(nczp::paged_join<16>), "paged_join<16>", 0, 0, 0, 0, {}},
    {reinterpret_cast<const void *>(nczp::paged_join<32>), "paged_join<32>", 0, 0, 0, 0, {}},
    {reinterpret_cast<const void *>(nczp::paged_join<64>), "paged_join<64>", 0, 0, 0, 0, {}},
    {reinterpret_cast<const void *>(nczp::paged_join<128>), "paged_join<128>", 0, 0, 0, 0, {}},
};
Kernel g_append[3] = {
    {reinterpret_cast<const void *>(nczp::paged_append<nczp::kF16, false>), "paged_append<copy>", 0, 0, 0, 0, {}},
    {reinterpret_cast<const void *>(nczp::paged_append<nczp::kF16, true>), "paged_append<f16,e4m3>", 0, 0, 0, 0, {}},
    {reinterpret_cast<const void *>(nczp::paged_append<nczp::kBF16, true>), "paged_append<bf16,e4m3>", 0, 0, 0, 0, {}},
};
Kernel g_plan = {reinterpret_cast<const void *>(nczp::paged_plan), "paged_plan", nczp::kPlanSmem, 0, 0, 0, {}};

template <class Fn>
void each_kernel(Fn fn) {
    for (auto &by_dim : g_decode)
        for (auto &by_rows : by_dim)
            for (Kernel &k : by_rows)
                if (k.fn != nullptr) fn(k);
    for (auto &by_dim : g_few)
        for (auto &by_rows : by_dim)
            for (Kernel &k : by_rows)
                if (k.fn != nullptr) fn(k);
    for (auto &by_dim : g_wide)
        for (auto &by_rows : by_dim)
            for (Kernel &k : by_rows) fn(k);
    for (Kernel &k : g_join) fn(k);
    for (Kernel &k : g_append) fn(k);
    fn(g_plan);
}

int device_sms(int dev) {
    std::lock_guard<std::mutex> lock(g_mu);
    if (g_sms[dev] == 0) {
        int n = 0;
        if (drv().sm_count(dev, &n) != cudaSuccess || n <= 0) n = 148;
        g_sms[dev] = n;
    }
    return g_sms[dev];
}

// Launches on the current device `dev`.
int launch(Kernel &k, unsigned grid, unsigned block, int dev, void *stream, void **args) {
    if (k.smem > 0) {
        std::lock_guard<std::mutex> lock(g_mu);
        if (!k.ready[dev]) {
            const int e = drv().set_max_dynamic_smem(k.fn, k.smem);
            if (e != cudaSuccess) return map_cuda_error(e);
            k.ready[dev] = true;
        }
    }
    const int e = drv().launch_kernel(k.fn, grid, block, static_cast<size_t>(k.smem), stream, args);
    if (e != cudaSuccess) return map_cuda_error(e);
    ncz::count_launch();
    return NCZ_SUCCESS;
}

// Runs fn(device) with `device` (-1 = current) current, then restores the caller's.
template <class Fn>
int on_device(int device, Fn fn) {
    int prev = 0;
    int e = drv().get_device(&prev);
    if (e != cudaSuccess) return map_cuda_error(e);
    const int dev = device >= 0 ? device : prev;
    if (dev < 0 || dev >= kMaxDevices) return NCZ_ERROR_INVALID_DEVICE;
    if (dev != prev && (e = drv().set_device(dev)) != cudaSuccess) return map_cuda_error(e);
    const int st = fn(dev);
    if (dev != prev) drv().set_device(prev);
    return st;
}

bool aligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

nczp::FastDiv fast_div(uint32_t d) {
    uint32_t s = 0;
    while ((uint64_t(1) << s) < d) ++s;
    const uint64_t mul = ((uint64_t(1) << 32) * ((uint64_t(1) << s) - d)) / d + 1;
    return {d, static_cast<uint32_t>(mul), s};
}

// Whether rows of `row` elements at i0 * st[0] + i1 * st[1] + i2 * st[2], i < n, keep apart.
bool rows_apart(size_t row, std::initializer_list<std::pair<size_t, size_t>> dims) {
    std::pair<size_t, size_t> d[3];  // stride, count
    size_t used = 0;
    for (const auto &x : dims)
        if (x.second > 1) d[used++] = x;
    std::sort(d, d + used);
    size_t span = row;  // elements the dimensions so far reach over
    for (size_t i = 0; i < used; ++i) {
        if (d[i].first < span) return false;
        span += (d[i].second - 1) * d[i].first;
    }
    return true;
}

int element_size(int dtype) { return dtype == NCZ_DTYPE_E4M3 ? 1 : dtype == NCZ_DTYPE_F32 ? 4 : 2; }

int check_cache(const ncz_paged_cache *c) {
    if (c == nullptr || c->k == nullptr || c->v == nullptr) return NCZ_ERROR_INVALID_VALUE;
    if (c->dtype != NCZ_DTYPE_F16 && c->dtype != NCZ_DTYPE_BF16 && c->dtype != NCZ_DTYPE_E4M3)
        return NCZ_ERROR_INVALID_VALUE;
    const size_t d = c->head_dim;
    if (d != 16 && d != 32 && d != 64 && d != 128) return NCZ_ERROR_INVALID_VALUE;
    if (d == 16 && c->dtype == NCZ_DTYPE_E4M3) return NCZ_ERROR_INVALID_VALUE;
    if (c->dtype != NCZ_DTYPE_E4M3 && (c->k_scale != nullptr || c->v_scale != nullptr)) return NCZ_ERROR_INVALID_VALUE;
    if (c->num_pages == 0 || c->page_size == 0 || c->kv_heads == 0) return NCZ_ERROR_INVALID_VALUE;
    if (c->num_pages > kMaxInt || c->page_size > kMaxInt || c->kv_heads > 65536) return NCZ_ERROR_INVALID_VALUE;
    const size_t strides[6] = {c->k_page_stride, c->k_token_stride, c->k_head_stride,
                               c->v_page_stride, c->v_token_stride, c->v_head_stride};
    for (const size_t s : strides)
        if (s > kMaxStride) return NCZ_ERROR_OVERFLOW;
    const size_t el = static_cast<size_t>(element_size(c->dtype));
    const size_t counts[3] = {c->num_pages, c->page_size, c->kv_heads};
    for (int i = 0; i < 6; i += 3) {
        // The last element's offset in bytes must stay inside 63 bits.
        unsigned __int128 reach = d;
        for (int j = 0; j < 3; ++j)
            reach += static_cast<unsigned __int128>(counts[j] - 1) * strides[i + j];
        if (reach * el > (static_cast<unsigned __int128>(1) << 62)) return NCZ_ERROR_OVERFLOW;
        if (!rows_apart(d, {{strides[i], counts[0]}, {strides[i + 1], counts[1]}, {strides[i + 2], counts[2]}}))
            return NCZ_ERROR_INVALID_VALUE;
    }
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return NCZ_ERROR_MISALIGNED;
    for (int i = 0; i < 6; ++i)
        if (counts[i % 3] > 1 && strides[i] * el % 16 != 0) return NCZ_ERROR_MISALIGNED;
    return NCZ_SUCCESS;
}

// Query heads of one item / 8 as a power: 8, 16 or 32 heads share one pass
// over the keys; larger groups read them once per 32 heads.
int rows_index(size_t group) { return group <= 8 ? 0 : group <= 16 ? 1 : 2; }

int dim_index(size_t d) { return d == 16 ? 0 : d == 32 ? 1 : d == 64 ? 2 : 3; }

// The kernel of a call and the query heads of its items.
struct Choice {
    Kernel *kernel;
    int rows;
};

Choice narrow_choice(const ncz_paged_cache &c, size_t group) {
    const int i = rows_index(group);
    return {&g_decode[c.dtype - 1][dim_index(c.head_dim)][i], 8 << i};
}

// Whether the tcgen05 kernel exists for a cache and pays for a group of query
// heads: from 17 on (batch 16, 4 K/V heads, 8192 keys, head_dim 64: 16 query heads
// 38.7 us with the warp MMAs and 40.1 us with it, 24: 55.8 and 40.6), at
// head_dim 128 from 9 on (12: 59.6 and 56.3, 32: 86.5 and 58.5; 8: 50.2 and 55.6).
bool has_wide(const ncz_paged_cache &c, size_t group) {
    return c.dtype != NCZ_DTYPE_E4M3 && c.head_dim >= 64 && group >= (c.head_dim == 128 ? 9 : 17);
}

Choice wide_choice(const ncz_paged_cache &c, size_t group) {
    const int i = group <= 32 ? 0 : group <= 64 ? 1 : 2;
    return {&g_wide[c.dtype == NCZ_DTYPE_BF16][c.head_dim == 128][i], 32 << i};
}

// The kernel of a call over up to `keys` keys a request.  f32 outputs stay with
// the warp MMAs: those sums are added in f32 every step, while tensor memory
// accumulates (and cuts off) over a row's whole length.  So do small launches:
// the tcgen05 kernel takes 128 keys a step and starts and ends slower (32 query
// heads of 8 K/V heads, head_dim 128: one request of 2000 keys, 128 steps in all,
// 14.4 us with the warp MMAs and 15.0 us with it, of 8000 keys 23.6 and 19.3;
// 64 requests of 300 keys, 3 steps each, 46.1 and 52.4, of 1000 keys 92.0 and 73.2).  So does a scale of
// 0, which takes a Q of its own (nczp::times_zero16): the registers for that cost the
// tcgen05 kernel up to 8 % of every other launch.
Choice choose(const ncz_paged_cache &c, size_t group, int o_dtype, float scale_log2, size_t batch, size_t keys, int sms) {
    const Choice narrow = narrow_choice(c, group);
    if (!has_wide(c, group) || o_dtype == NCZ_DTYPE_F32 || scale_log2 == 0.0f) return narrow;
    const Choice wide = wide_choice(c, group);
    const size_t each = (keys + nczp::kWideTile - 1) / nczp::kWideTile, blocks = (group + wide.rows - 1) / wide.rows;
    const size_t total = batch * c.kv_heads * blocks * each, longest = std::min(each, total / sms + 1);
    // Tensor memory's sums lose up to 7e-8 of themselves a step (measured over 80000 steps): at most a
    // seventh of the rounding of o over this many steps of a row in one CTA.
    const size_t limit = o_dtype == NCZ_DTYPE_F16 ? 1024 : 8192;
    return each >= 4 && total >= 2 * static_cast<size_t>(sms) && longest <= limit ? wide : narrow;
}

// CTAs of a launch at most: what is resident at once.
int max_ctas(const Kernel &k, int sms) { return sms * k.ctas; }

// Whether a cluster of eight CTAs per item is taken (paged_decode_few): the clusters are resident at
// once, and a CTA's run of tiles is at most two, and a quarter, longer than the even share that
// paged_decode would give it, which the join it saves pays for.  Eight rows (8 K/V heads), head_dim 128 bf16:
// 300 keys 8.1 -> 6.0 us, 1000 8.4 -> 7.0, 2000 9.0 -> 8.9, 4000 10.0 and 12.5; 32 rows: 500 keys
// 10.2 -> 6.8, 4000 21.5 -> 17.8; 64 rows of 500 keys (two waves of clusters) 11.3 and 12.4.
bool few_rows(size_t items, size_t most, size_t ctas, int sms) {
    const size_t run = (most + nczp::kDecodeCluster - 1) / nczp::kDecodeCluster, even = (items * most + ctas - 1) / ctas;
    return most > 1 && items * nczp::kDecodeCluster <= 2 * static_cast<size_t>(sms) && run <= 2 + even + even / 4;
}

size_t records_bytes(int ctas) { return (static_cast<size_t>(ctas) * sizeof(int4) + 255) / 256 * 256; }

size_t workspace_need(const Kernel &k, size_t d, int rows, int sms) {
    const size_t ctas = static_cast<size_t>(max_ctas(k, sms));
    return records_bytes(static_cast<int>(ctas)) + 2 * ctas * rows * (d * sizeof(float) + sizeof(float2));
}

int check_heads(const ncz_paged_cache &c, size_t q_heads) {
    if (q_heads == 0 || q_heads > 65536 || q_heads % c.kv_heads != 0) return NCZ_ERROR_INVALID_VALUE;
    return NCZ_SUCCESS;
}

// Whether a launch's CTAs each stay with one head block (nczp::paged_decode's by_head).
bool choose_by_head(size_t head_blocks, size_t ctas) {
    return head_blocks > 1 && head_blocks <= ctas && (ctas % head_blocks) * 16 <= ctas;
}

}  // namespace

extern "C" {

int ncz_paged_validate(const ncz_paged_cache *cache) { return check_cache(cache); }

int ncz_paged_plan(const ncz_paged_plan_desc *desc) {
    if (desc == nullptr) return NCZ_ERROR_INVALID_VALUE;
    const ncz_paged_plan_desc &d = *desc;
    if (d.free_count == nullptr || d.left == nullptr) return NCZ_ERROR_INVALID_VALUE;
    if (d.requests > 0 && (d.held == nullptr || d.added == nullptr || d.seq_lens == nullptr ||
                           (d.block_table == nullptr && d.table_width > 0)))
        return NCZ_ERROR_INVALID_VALUE;
    if (d.free_capacity > 0 && d.free_pages == nullptr) return NCZ_ERROR_INVALID_VALUE;
    if (d.slot_capacity > 0 && d.slots == nullptr) return NCZ_ERROR_INVALID_VALUE;
    if (d.page_size == 0 || d.page_size > kMaxInt) return NCZ_ERROR_INVALID_VALUE;
    if (d.requests > kMaxRequests || d.free_capacity > kMaxInt || d.slot_capacity > kMaxInt || d.table_width > kMaxInt)
        return NCZ_ERROR_INVALID_VALUE;
    if (d.table_width * d.page_size > kMaxInt) return NCZ_ERROR_OVERFLOW;  // positions are 32-bit
    if (d.table_stride > kMaxStride / 2) return NCZ_ERROR_OVERFLOW;
    if (d.requests > 1 && d.table_stride < d.table_width) return NCZ_ERROR_INVALID_VALUE;
    for (const void *x : {static_cast<const void *>(d.held), static_cast<const void *>(d.added),
                          static_cast<const void *>(d.free_pages), static_cast<const void *>(d.free_count),
                          static_cast<const void *>(d.block_table), static_cast<const void *>(d.seq_lens),
                          static_cast<const void *>(d.positions), static_cast<const void *>(d.starts),
                          static_cast<const void *>(d.left), static_cast<const void *>(d.status)})
        if (!aligned(x, 4)) return NCZ_ERROR_MISALIGNED;
    if (!aligned(d.slots, 8)) return NCZ_ERROR_MISALIGNED;
    // seq_lens is `held` or apart from it, and apart from `added`.
    auto overlap = [&](const int32_t *a) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(d.seq_lens);
        return x < y + 4 * d.requests && y < x + 4 * d.requests;
    };
    if (d.requests > 0 && ((d.held != d.seq_lens && overlap(d.held)) || overlap(d.added))) return NCZ_ERROR_INVALID_VALUE;
    nczp::PlanParams p{};
    p.held = d.held;
    p.added = d.added;
    p.free_pages = d.free_pages;
    p.free_count = d.free_count;
    p.table = d.block_table;
    p.seq_lens = d.seq_lens;
    p.slots = reinterpret_cast<long long *>(d.slots);
    p.positions = d.positions;
    p.starts = d.starts;
    p.left = d.left;
    p.status = d.status;
    p.table_stride = static_cast<long long>(d.table_stride);
    p.slot_capacity = static_cast<long long>(d.slot_capacity);
    p.requests = static_cast<int>(d.requests);
    p.width = static_cast<int>(d.table_width);
    p.free_capacity = static_cast<int>(d.free_capacity);
    p.page = fast_div(static_cast<uint32_t>(d.page_size));
    // A cluster per 4096 slots, up to what an SM count of 148 holds at once, unless outputs are
    // in place of inputs that another cluster may not have read.
    const bool in_place = d.held == d.seq_lens || d.free_count == d.left;
    const unsigned clusters =
        in_place ? 1u : static_cast<unsigned>(std::min<size_t>(kPlanClusters, 1 + d.slot_capacity / kSlotsPerCluster));
    return on_device(d.device, [&](int dev) {
        void *args[1] = {&p};
        return launch(g_plan, nczp::kPlanCluster * clusters, nczp::kPlanThreads, dev, d.stream, args);
    });
}

int ncz_paged_append(const ncz_paged_cache *cache, const ncz_paged_append_desc *desc) {
    int st = check_cache(cache);
    if (st != NCZ_SUCCESS) return st;
    if (desc == nullptr) return NCZ_ERROR_INVALID_VALUE;
    const ncz_paged_cache &c = *cache;
    const ncz_paged_append_desc &d = *desc;
    if (d.in_dtype != NCZ_DTYPE_F16 && d.in_dtype != NCZ_DTYPE_BF16) return NCZ_ERROR_INVALID_VALUE;
    if (c.dtype != NCZ_DTYPE_E4M3 && c.dtype != d.in_dtype) return NCZ_ERROR_INVALID_VALUE;
    if (d.tokens == 0) return NCZ_SUCCESS;
    if (d.k == nullptr || d.v == nullptr || d.slots == nullptr || d.tokens > kMaxInt) return NCZ_ERROR_INVALID_VALUE;
    if (c.k == c.v) return NCZ_ERROR_INVALID_VALUE;  // each slot would take both rows
    if (!aligned(d.k, 2) || !aligned(d.v, 2) || !aligned(d.slots, 8)) return NCZ_ERROR_MISALIGNED;
    for (const size_t s : {d.k_token_stride, d.k_head_stride, d.v_token_stride, d.v_head_stride})
        if (s > kMaxStride / 4) return NCZ_ERROR_OVERFLOW;
    const long long el = element_size(c.dtype);
    nczp::AppendParams p{};
    p.k = static_cast<const char *>(d.k);
    p.v = static_cast<const char *>(d.v);
    p.ck = static_cast<char *>(c.k);
    p.cv = static_cast<char *>(c.v);
    p.k_scale = c.k_scale;
    p.v_scale = c.v_scale;
    p.slots = reinterpret_cast<const long long *>(d.slots);
    p.k_tok = static_cast<long long>(d.k_token_stride) * 2;
    p.k_head = static_cast<long long>(d.k_head_stride) * 2;
    p.v_tok = static_cast<long long>(d.v_token_stride) * 2;
    p.v_head = static_cast<long long>(d.v_head_stride) * 2;
    p.ck_page = static_cast<long long>(c.k_page_stride) * el;
    p.ck_tok = static_cast<long long>(c.k_token_stride) * el;
    p.ck_head = static_cast<long long>(c.k_head_stride) * el;
    p.cv_page = static_cast<long long>(c.v_page_stride) * el;
    p.cv_tok = static_cast<long long>(c.v_token_stride) * el;
    p.cv_head = static_cast<long long>(c.v_head_stride) * el;
    p.tokens = static_cast<long long>(d.tokens);
    p.num_slots = static_cast<long long>(c.num_pages) * static_cast<long long>(c.page_size);
    p.head_pieces = static_cast<int>(c.head_dim / nczp::kAppendPiece);
    p.pieces = static_cast<int>(c.kv_heads) * p.head_pieces;
    p.group = std::max(1, nczp::kAppendThreads / p.pieces);
    p.vec = aligned(d.k, 16) && aligned(d.v, 16) && p.k_tok % 16 == 0 && p.k_head % 16 == 0 && p.v_tok % 16 == 0 &&
            p.v_head % 16 == 0;
    p.page_size = static_cast<uint32_t>(c.page_size);
    const long long blocks = (p.tokens + p.group - 1) / p.group;
    Kernel &k = g_append[c.dtype != NCZ_DTYPE_E4M3 ? 0 : d.in_dtype == NCZ_DTYPE_F16 ? 1 : 2];
    return on_device(d.device, [&](int dev) {
        void *args[1] = {&p};
        return launch(k, static_cast<unsigned>(blocks), nczp::kAppendThreads, dev, d.stream, args);
    });
}

int ncz_paged_decode_workspace(const ncz_paged_cache *cache, size_t q_heads, int device, size_t *bytes) {
    int st = check_cache(cache);
    if (st != NCZ_SUCCESS) return st;
    if (bytes == nullptr) return NCZ_ERROR_INVALID_VALUE;
    st = check_heads(*cache, q_heads);
    if (st != NCZ_SUCCESS) return st;
    const size_t group = q_heads / cache->kv_heads;
    return on_device(device, [&](int dev) {
        // For any batch and output type: the larger of the kernels that may be taken.
        const Choice narrow = narrow_choice(*cache, group);
        *bytes = workspace_need(*narrow.kernel, cache->head_dim, narrow.rows, device_sms(dev));
        if (has_wide(*cache, group)) {
            const Choice wide = wide_choice(*cache, group);
            *bytes = std::max(*bytes, workspace_need(*wide.kernel, cache->head_dim, wide.rows, device_sms(dev)));
        }
        return NCZ_SUCCESS;
    });
}

int ncz_paged_decode(const ncz_paged_cache *cache, const ncz_paged_decode_desc *desc) {
    int st = check_cache(cache);
    if (st != NCZ_SUCCESS) return st;
    if (desc == nullptr) return NCZ_ERROR_INVALID_VALUE;
    const ncz_paged_cache &c = *cache;
    const ncz_paged_decode_desc &d = *desc;
    st = check_heads(c, d.q_heads);
    if (st != NCZ_SUCCESS) return st;
    if (d.q_dtype != NCZ_DTYPE_F16 && d.q_dtype != NCZ_DTYPE_BF16) return NCZ_ERROR_INVALID_VALUE;
    if (c.dtype != NCZ_DTYPE_E4M3 && c.dtype != d.q_dtype) return NCZ_ERROR_INVALID_VALUE;
    if (d.o_dtype != NCZ_DTYPE_F32 && d.o_dtype != NCZ_DTYPE_F16 && d.o_dtype != NCZ_DTYPE_BF16)
        return NCZ_ERROR_INVALID_VALUE;
    if (d.batch == 0) return NCZ_SUCCESS;
    if (d.q == nullptr || d.o == nullptr || d.seq_lens == nullptr || (d.block_table == nullptr && d.table_width > 0))
        return NCZ_ERROR_INVALID_VALUE;
    // q is read while o and lse are written.
    if (d.o == d.q || d.lse == d.q || d.lse == d.o) return NCZ_ERROR_INVALID_VALUE;
    if (d.batch > kMaxRequests || d.table_width > kMaxInt) return NCZ_ERROR_INVALID_VALUE;
    if (d.table_width * c.page_size > kMaxInt) return NCZ_ERROR_OVERFLOW;
    for (const size_t s : {d.q_batch_stride, d.q_head_stride, d.o_batch_stride, d.o_head_stride, d.table_stride})
        if (s > kMaxStride / 4) return NCZ_ERROR_OVERFLOW;
    if (d.batch > 1 && d.table_stride < d.table_width) return NCZ_ERROR_INVALID_VALUE;
    if (!rows_apart(c.head_dim, {{d.o_batch_stride, d.batch}, {d.o_head_stride, d.q_heads}}))
        return NCZ_ERROR_INVALID_VALUE;
    const size_t o_size = static_cast<size_t>(element_size(d.o_dtype));
    if (!aligned(d.q, 2) || !aligned(d.o, o_size) || !aligned(d.lse, 4) || !aligned(d.block_table, 4) ||
        !aligned(d.seq_lens, 4))
        return NCZ_ERROR_MISALIGNED;
    const size_t group = d.q_heads / c.kv_heads;
    nczp::DecodeParams p{};
    p.q = static_cast<const char *>(d.q);
    p.k = static_cast<const char *>(c.k);
    p.v = static_cast<const char *>(c.v);
    p.o = d.o;
    p.lse = d.lse;
    p.k_scale = c.k_scale;
    p.v_scale = c.v_scale;
    p.table = d.block_table;
    p.lens = d.seq_lens;
    const long long el = element_size(c.dtype);
    p.k_page = static_cast<long long>(c.k_page_stride) * el;
    p.k_tok = static_cast<long long>(c.k_token_stride) * el;
    p.k_head = static_cast<long long>(c.k_head_stride) * el;
    p.v_page = static_cast<long long>(c.v_page_stride) * el;
    p.v_tok = static_cast<long long>(c.v_token_stride) * el;
    p.v_head = static_cast<long long>(c.v_head_stride) * el;
    p.q_batch = static_cast<long long>(d.q_batch_stride);
    p.q_head = static_cast<long long>(d.q_head_stride);
    p.o_batch = static_cast<long long>(d.o_batch_stride);
    p.o_head = static_cast<long long>(d.o_head_stride);
    p.table_stride = static_cast<long long>(d.table_stride);
    p.batch = static_cast<int>(d.batch);
    p.group = static_cast<int>(group);
    p.width_keys = static_cast<int>(d.table_width * c.page_size);
    p.window = static_cast<int>(std::min(d.window, kMaxInt));
    p.num_pages = static_cast<int>(c.num_pages);
    p.page = fast_div(static_cast<uint32_t>(c.page_size));
    p.scale_log2 = static_cast<float>(static_cast<double>(d.scale) * 1.4426950408889634);
    p.whole_groups = c.page_size % 16 == 0;
    p.same_strides = p.k_page == p.v_page && p.k_tok == p.v_tok;
    p.q_bf16 = d.q_dtype == NCZ_DTYPE_BF16;
    p.o_dtype = d.o_dtype;
    p.q_vec = aligned(d.q, 8) && d.q_batch_stride % 4 == 0 && d.q_head_stride % 4 == 0;
    p.o_vec = aligned(d.o, 4 * o_size) && d.o_batch_stride % 4 == 0 && d.o_head_stride % 4 == 0;
    // 16-bit parts of P: f32 o takes the bits of f32 (3 of bf16, 2 of f16), 16-bit o two parts as
    // well.  One f16 part (2^-11 of a weight) is eight times finer than bf16 o (2^-8); for e4m3 K/V, where
    // the conversions keep the SM busy, a second one costs 2 % with 8 query heads a K/V head (16 requests of
    // 8192 keys, 4 K/V heads, head_dim 128: 33.6 and 34.3 us) and 8 % with 32 (69.3 and 74.8).
    // f16's smallest step is 2^-24 and a row's largest P 2^8 or more, so in f16 parts, however many, a
    // weight is also off by up to 2^-33 of the row's largest: that is the larger error below 2^-22 of
    // it with one part, below 2^-11 with two, and weights below 2^-33 are in the sum but not in o.
    p.p_parts = c.dtype == NCZ_DTYPE_BF16 && d.o_dtype == NCZ_DTYPE_F32 ? 3
                : c.dtype == NCZ_DTYPE_E4M3 && d.o_dtype == NCZ_DTYPE_BF16 ? 1 : 2;

    // Keys of a request at most: the lengths are on the device, the table's width bounds them.
    const size_t keys = d.window > 0 ? std::min(d.window, static_cast<size_t>(p.width_keys)) : p.width_keys;

    return on_device(d.device, [&](int dev) {
        const int sms = device_sms(dev);
        const Choice choice = choose(c, group, d.o_dtype, p.scale_log2, d.batch, keys, sms);
        Kernel &k = *choice.kernel;
        const int rows = choice.rows;
        const size_t blocks = (group + rows - 1) / rows;
        p.blocks = static_cast<int>(blocks);
        p.head_blocks = static_cast<int>(c.kv_heads * blocks);
        if (d.workspace == nullptr || d.workspace_bytes < workspace_need(k, c.head_dim, rows, sms))
            return static_cast<int>(NCZ_ERROR_OUT_OF_MEMORY);
        if (!aligned(d.workspace, 16)) return static_cast<int>(NCZ_ERROR_MISALIGNED);
        const size_t tile = static_cast<size_t>(k.tile);
        const size_t most = std::max<size_t>(1, (keys + (d.window > 0 ? 15 : 0) + tile - 1) / tile);
        const size_t items = d.batch * static_cast<size_t>(p.head_blocks);
        if (rows <= 16 && few_rows(items, most, static_cast<size_t>(max_ctas(k, sms)), sms)) {
            Kernel &few = g_few[c.dtype - 1][dim_index(c.head_dim)][rows == 16];
            void *args[1] = {&p};
            return launch(few, static_cast<unsigned>(items * nczp::kDecodeCluster), few.threads, dev, d.stream, args);
        }
        const int ctas = max_ctas(k, sms);
        unsigned grid = static_cast<unsigned>(
            most > static_cast<size_t>(ctas) ? ctas : std::min(static_cast<size_t>(ctas), most * items));
        p.by_head = choose_by_head(static_cast<size_t>(p.head_blocks), grid);
        if (p.by_head) grid -= grid % static_cast<unsigned>(p.head_blocks);
        p.records_by_item = items <= grid;
        p.ctas = static_cast<int>(grid);
        char *ws = static_cast<char *>(d.workspace);
        p.records = reinterpret_cast<int4 *>(ws);
        p.part_o = reinterpret_cast<float *>(ws + records_bytes(ctas));
        p.part_ml = reinterpret_cast<float2 *>(p.part_o + 2 * static_cast<size_t>(ctas) * rows * c.head_dim);
        void *args[1] = {&p};
        // Rows of one tile are whole in one CTA: nothing to join.
        if (most == 1) return launch(k, grid, k.threads, dev, d.stream, args);
        std::lock_guard<std::mutex> lock(pair_mutex(dev, d.stream));
        const int s = launch(k, grid, k.threads, dev, d.stream, args);
        if (s != NCZ_SUCCESS) return s;
        // Quads (four elements) per join block: as few as keep the grid within
        // four blocks an SM, a 128-byte line of a part's row at least.
        const unsigned records = p.records_by_item ? static_cast<unsigned>(items) : grid;
        const int total = static_cast<int>(std::min(group, static_cast<size_t>(rows)) * c.head_dim / 4);
        int quads = 8, join_rows = rows;
        auto blocks_of = [&](int q) { return (total + q - 1) / q; };
        while (quads < nczp::kJoinThreads &&
               static_cast<size_t>(records) * blocks_of(quads) > 4 * static_cast<size_t>(sms))
            quads *= 2;
        int per_record = blocks_of(quads);
        void *join_args[4] = {&p, &join_rows, &quads, &per_record};
        return launch(g_join[dim_index(c.head_dim)], records * per_record, nczp::kJoinThreads, dev, d.stream,
                      join_args);
    });
}

int ncz_paged_sync_status(int device) {
    return on_device(device, [](int) {
        uint32_t word = 0;
        const void *sym = static_cast<const void *>(&nczp::g_paged_status);
        int e = drv().device_synchronize();
        if (e == cudaSuccess) e = drv().symbol_read(&word, sym, sizeof(word));
        if (e == cudaSuccess && word != 0) {
            const uint32_t zero = 0;
            e = drv().symbol_write(sym, &zero, sizeof(zero));
        }
        if (e != cudaSuccess) return map_cuda_error(e);
        return static_cast<int>(word != 0 ? NCZ_ERROR_DEVICE_TIMEOUT : NCZ_SUCCESS);
    });
}

int ncz_paged_test_set_wait_limit(int device, uint64_t cycles) {
    const unsigned long long v = cycles != 0 ? cycles : nczp::kPagedWaitLimit;
    return on_device(device, [&](int) {
        return map_cuda_error(drv().symbol_write(static_cast<const void *>(&nczp::g_paged_wait_limit), &v, sizeof(v)));
    });
}

int ncz_paged_test_drop_scores(int device, int enable) {
    const int v = enable != 0;
    return on_device(device, [&](int) {
        return map_cuda_error(drv().symbol_write(static_cast<const void *>(&nczp::g_paged_test_drop), &v, sizeof(v)));
    });
}

int ncz_paged_test_leave_merge(int device, int enable) {
    const int v = enable != 0;
    return on_device(device, [&](int) {
        return map_cuda_error(drv().symbol_write(static_cast<const void *>(&nczp::g_paged_test_leave), &v, sizeof(v)));
    });
}

}  // extern "C"

namespace ncz {

void reset_paged_caches() {
    std::lock_guard<std::mutex> lock(g_mu);
    std::memset(g_sms, 0, sizeof(g_sms));
    each_kernel([](Kernel &k) { std::memset(k.ready, 0, sizeof(k.ready)); });
}

const char *paged_kernel_label(const void *kernel) {
    const char *label = nullptr;
    each_kernel([&](Kernel &k) {
        if (k.fn == kernel) label = k.label;
    });
    return label;
}

// The join starts while the decode kernel's last CTAs still run (its blocks
// wait for their writes).
bool overlaps_predecessor(const void *kernel) {
    for (const Kernel &k : g_join)
        if (k.fn == kernel) return true;
    return false;
}

}  // namespace ncz
