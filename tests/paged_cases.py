"""Problems and 64-bit oracles for the paged-cache tests: numpy for plan, torch
float64 for append and decode, written from the definitions in
include/ncz_paged.h.  Nothing here needs a GPU."""
import math

import numpy as np
import torch

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def half_step(dtype):
    """Largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------- plan

def plan_oracle(held, added, free_pages, free_count, table, page, capacity):
    """Request by request; returns the outputs as a dict (table is copied)."""
    table = table.copy()
    n, width = table.shape
    free_count = min(max(int(free_count), 0), len(free_pages))
    seq_lens = held.copy()
    starts = np.zeros(n + 1, np.int64)
    slots, positions = [], []
    asked = taken = refused = 0
    for r in range(n):
        h, a = int(held[r]), int(added[r])
        tokens = max(a, 0)
        starts[r + 1] = starts[r] + tokens
        have = -(-max(h, 0) // page)
        want = -(-(max(h, 0) + tokens) // page)
        fits = h >= 0 and a >= 0 and want <= width
        need = want - have if fits else 0
        served = fits and (need == 0 or asked + need <= free_count)
        if served:
            for i in range(need):
                table[r, have + i] = free_pages[free_count - 1 - asked - i]
            if need:
                taken = asked + need
            seq_lens[r] = h + a
        else:
            refused += 1
        asked += need
        for j in range(tokens):
            if len(slots) >= capacity:
                break
            position = max(h, 0) + j
            page_id = int(table[r, position // page]) if served else -1
            slots.append(page_id * page + position % page if page_id >= 0 else -1)
            positions.append(min(position, 2**31 - 1))
    pad = capacity - len(slots)
    total = int(starts[n])
    return {"block_table": table, "seq_lens": seq_lens, "slots": np.array(slots + [-1] * pad, np.int64),
            "positions": np.array(positions + [0] * pad, np.int64), "starts": np.minimum(starts, capacity),
            "left": np.array([free_count - taken]),
            "status": np.array([total, taken, refused, max(0, total - capacity)])}


# ---------------------------------------------------------------- decode

def decode_oracle(q, k_pages, v_pages, table, lens, scale, window=0, k_scale=None, v_scale=None, p_step=2.0 ** -17):
    """(o, lse, tol_o, tol_lse) in float64 from CPU tensors.  The tolerances bound
    a kernel that keeps scores, softmax and sums in f32:

    score of a key: products of 16-bit values are exact, D of them are summed in
    f32 (each addition off by at most 2^-23 of the sum of magnitudes a, in any
    order and with truncation), then scaled, offset and put through a
    base-2 exponential (2^-22): ds = (D 2^-23 a + 2^-21 |s|) + 2^-22;
    sums over n keys: at most 2 n / 16 + 64 additions in a chain, each off by 2^-23;
    P in two bf16 parts (16 bits): 2^-17; `p_step`, where P is given fewer (one f16 part for
    e4m3 K/V with bf16 o: each weight is off by at most 2^-11 of it, so o by 2^-11 of sum p |v| / l).
    An o is a ratio of two such sums: twice that, of sum p |v| / l."""
    batch, heads, dim = q.shape
    kv = k_pages.shape[2]
    page, pages = k_pages.shape[1], k_pages.shape[0]
    group = heads // kv
    k_all, v_all = k_pages.float(), v_pages.float()
    o = torch.zeros(batch, heads, dim, dtype=torch.float64)
    lse = torch.full((batch, heads), -math.inf, dtype=torch.float64)
    tol_o, tol_lse = torch.zeros_like(o), torch.zeros_like(lse)
    for b in range(batch):
        n = min(max(int(lens[b]), 0), table.shape[1] * page)
        lo = max(0, n - window) if window else 0
        keys = [(int(table[b, j // page]), j % page) for j in range(lo, n)]
        keys = [(p, r) for p, r in keys if 0 <= p < pages]
        if not keys:
            continue
        at = torch.tensor(keys)
        for h in range(heads):
            g = h // group
            k, v = (x[at[:, 0], at[:, 1], g].double() for x in (k_all, v_all))
            if k_scale is not None:
                k = k * float(k_scale[g])
            if v_scale is not None:
                v = v * float(v_scale[g])
            x = q[b, h].double()
            s = k @ x * scale
            lse[b, h] = torch.logsumexp(s, 0)
            p = torch.softmax(s, 0)
            o[b, h] = p @ v
            magnitude = float((k.abs() @ x.abs() * abs(scale)).max())
            ds = dim * 2.0 ** -23 * magnitude + 2.0 ** -21 * float(s.abs().max()) + 2.0 ** -22
            sums = (2 * len(keys) / 16 + 64) * 2.0 ** -23
            tol_o[b, h] = (2 * (ds + sums) + max(p_step, 2.0 ** -16)) * (p @ v.abs())
            tol_lse[b, h] = ds + sums + 2.0 ** -22 * abs(float(lse[b, h]))
    return o, lse, tol_o, tol_lse


def decode_problem(batch, q_heads, kv_heads, dim, page, lens, dtype, *, cache_dtype=None, seed=0, extra_pages=3,
                   width=None, fill=float("nan")):
    """CPU tensors of a decode problem: pages in random order; rows that no
    request's length covers hold `fill`, NaN unless told otherwise, and the
    table's unused entries name such pages."""
    g = torch.Generator().manual_seed(seed)
    cache_dtype = cache_dtype or dtype
    have = [-(-n // page) for n in lens]
    pages = sum(have) + extra_pages
    width = width or max(1, max(have) + 1)
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((batch, width), order[-1], dtype=torch.int32)
    shape = (pages, page, kv_heads, dim)
    live = torch.zeros(pages, page, dtype=torch.bool)
    used = 0
    for b, n in enumerate(lens):
        for i in range(have[b]):
            table[b, i] = order[used]
            live[order[used], :min(page, n - i * page)] = True
            used += 1
    q = torch.randn(batch, q_heads, dim, generator=g).to(dtype)
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=g)
        if cache_dtype == E4M3:
            x = (x * 24).clamp(-448, 448)
        x = torch.where(live[:, :, None, None], x, torch.tensor(fill))
        out.append(x.to(cache_dtype))
    return {"q": q, "k": out[0], "v": out[1], "table": table, "lens": torch.tensor(lens, dtype=torch.int32),
            "scale": dim ** -0.5}
