"""The paged-cache operators on the GPU against 64-bit oracles
(tests/paged_cases.py).  plan and same-type append are compared exactly, decode
within the rounding bounds that the oracle derives."""
import math

import numpy as np
import pytest

from tests import paged_cases as P

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

F32, F16, BF16, E4M3 = P.F32, P.F16, P.BF16, P.E4M3


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- plan

def run_plan(ncz, held, added, free_pages, free_count, table, page, capacity, *, in_place=False, stream=None):
    n = len(held)
    t = {"held": i32(held), "added": i32(added), "free": i32(free_pages), "count": i32([free_count]),
         "table": i32(table).view(n, -1)}
    made = lambda k, dt=torch.int32: torch.full((k,), -77, dtype=dt, device="cuda")  # noqa: E731
    out = {"block_table": t["table"], "seq_lens": t["held"] if in_place else made(n),
           "slots": made(capacity, torch.int64), "positions": made(capacity), "starts": made(n + 1),
           "left": t["count"] if in_place else made(1), "status": made(4)}
    ncz.paged.plan(t["held"], t["added"], t["free"], t["count"], t["table"], out["seq_lens"], out["slots"],
                   page_size=page, positions=out["positions"], starts=out["starts"],
                   left=None if in_place else out["left"], status=out["status"], stream=stream)
    torch.cuda.synchronize()
    return {k: v.cpu().numpy() for k, v in out.items()}


def plan_problem(n, page, width, held_hi, added_hi, spare, seed):
    rng = np.random.default_rng(seed)
    held = rng.integers(0, held_hi + 1, n).astype(np.int32)
    added = rng.integers(0, added_hi + 1, n).astype(np.int32)
    have = -(-held // page)
    need = np.maximum(-(-(held + added) // page) - have, 0)
    ids = rng.permutation(int(have.sum()) + int(need.sum()) + max(spare, 0)).astype(np.int32)
    table = np.full((n, width), -5, np.int32)
    at = 0
    for r in range(n):
        k = min(int(have[r]), width)
        table[r, :k] = ids[at:at + k]
        at += k
    free = ids[at:]
    count = len(free) + min(spare, 0)
    return held, added, free, count, table, int(added.sum())


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,page,held_hi,added_hi,spare", [
    (1, 16, 0, 1, 0), (1, 1, 3, 9, 2), (33, 7, 50, 1, 4), (256, 16, 400, 1, 9), (100, 5, 0, 60, 0), (64, 128, 90, 300, 1),
    (4096, 16, 40, 2, 3), (4097, 3, 9, 3, 0), (9000, 32, 64, 5, -40), (300, 8, 30, 20, -200), (5, 1000, 0, 30000, 7),
])
def test_plan_matches_oracle(ncz, n, page, held_hi, added_hi, spare, in_place):
    width = -(-(held_hi + added_hi) // page) + 2
    held, added, free, count, table, total = plan_problem(n, page, width, held_hi, added_hi, spare, n + page)
    for capacity in (total + 13, max(0, total - 3)):
        want = P.plan_oracle(held, added, free, count, table, page, capacity)
        got = run_plan(ncz, held, added, free, count, table, page, capacity, in_place=in_place)
        for name in want:
            assert np.array_equal(got[name], want[name]), (name, capacity)
    if spare < 0:
        assert want["status"][2] > 0


def test_plan_refuses_bad_lengths_rows_and_counts(ncz):
    """Negative lengths, rows past the table's width, a free count past or below
    the stack, negative held page ids: refused requests, never a bad access."""
    big = 2**31 - 1
    held = np.array([-4, 5, big, 0, 30, 3, 40, 0], np.int32)
    added = np.array([3, -2, big, 33, 2, 4, 1, 0], np.int32)
    table = np.arange(8 * 5, dtype=np.int32).reshape(8, 5) + 1000
    table[5, 0] = -1
    free = np.arange(6, dtype=np.int32) + 7
    # big + big tokens would fill the slots: they are only counted, 100 of them kept
    for count in (6, 100, -3, big, 2):
        want = P.plan_oracle(held, np.minimum(added, 200), free, count, table, 8, 100)
        got = run_plan(ncz, held, np.minimum(added, 200), free, count, table, 8, 100)
        for name in want:
            assert np.array_equal(got[name], want[name]), (name, count)
    got = run_plan(ncz, held, added, free, 6, table, 8, 100)
    assert got["status"][0] == big and (got["slots"][:3] == -1).all() and got["starts"].max() == 100


def test_plan_of_no_requests_and_no_slots(ncz):
    made = lambda k, dt=torch.int32: torch.full((k,), -77, dtype=dt, device="cuda")  # noqa: E731
    none, count = made(0), i32([4])
    slots, starts, status = made(3, torch.int64), made(1), made(4)
    ncz.paged.plan(none, none, i32([1, 2, 3, 4]), count, none.view(0, 1), none, slots, page_size=4, starts=starts,
                   status=status)
    assert slots.tolist() == [-1] * 3 and starts.tolist() == [0] and status.tolist() == [0] * 4 and count.tolist() == [4]
    table = i32([[-1, -1]])
    ncz.paged.plan(i32([0]), i32([5]), i32([1, 2, 3, 4]), count, table, made(1), made(0, torch.int64), page_size=4)
    assert table.tolist() == [[4, 3]] and count.tolist() == [2]


def test_plan_strided_table_leaves_the_rest(ncz):
    held, added, free, count, table, total = plan_problem(20, 4, 6, 10, 10, 3, 1)
    wide = torch.full((25, 11), 99, dtype=torch.int32, device="cuda")
    view = wide[2:22, 3:9]
    view.copy_(i32(table))
    made = lambda k, dt=torch.int32: torch.full((k,), -77, dtype=dt, device="cuda")  # noqa: E731
    ncz.paged.plan(i32(held), i32(added), i32(free), i32([count]), view, made(20), made(total, torch.int64), page_size=4)
    want = P.plan_oracle(held, added, free, count, table, 4, total)
    assert np.array_equal(view.cpu().numpy(), want["block_table"])
    view.fill_(99)
    assert bool((wide == 99).all())


# ---------------------------------------------------------------- append

def pages_of(pages, page, kv, dim, dtype, layout):
    if layout == "heads_first":
        return torch.full((pages, kv, page, dim), 3.0, device="cuda").to(dtype).transpose(1, 2)
    if layout == "padded":
        return torch.full((pages, page, kv, dim + 16), 3.0, device="cuda").to(dtype)[..., :dim]
    return torch.full((pages, page, kv, dim), 3.0, device="cuda").to(dtype)


def rows_of(tokens, kv, dim, dtype, kind, g):
    if kind == "interleaved":  # K and V in one matrix, 16-byte rows
        x = torch.randn(tokens, 2 * kv, dim, generator=g, device="cuda").to(dtype)
        return x[:, :kv], x[:, kv:]
    if kind == "odd":          # rows that start on odd elements
        x = torch.randn(tokens, 2 * kv, dim + 1, generator=g, device="cuda").to(dtype)
        return x[:, :kv, 1:], x[:, kv:, 1:]
    if kind == "broadcast":    # one row for every head
        x = torch.randn(tokens, 2, 1, dim, generator=g, device="cuda").to(dtype)
        return x[:, 0].expand(tokens, kv, dim), x[:, 1].expand(tokens, kv, dim)
    return tuple(torch.randn(tokens, kv, dim, generator=g, device="cuda").to(dtype) for _ in range(2))


@pytest.mark.parametrize("layout,kind", [("plain", "plain"), ("heads_first", "interleaved"), ("padded", "odd"),
                                         ("plain", "broadcast")])
@pytest.mark.parametrize("tokens,kv,dim,page", [(1, 1, 16, 1), (5, 3, 32, 7), (700, 8, 128, 16), (333, 2, 64, 100)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_copies_rows_exactly(ncz, tokens, kv, dim, page, dtype, layout, kind):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    pages = tokens // page + 5
    k_pages, v_pages = (pages_of(pages, page, kv, dim, dtype, layout) for _ in range(2))
    k, v = rows_of(tokens, kv, dim, dtype, kind, g)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[tokens // 2] = -1
    if tokens > 3:
        slots[1] = pages * page          # past the cache: skipped, like any slot outside it
        slots[2] = -(1 << 40)
        slots[3] = 1 << 62
    want = [x.clone() for x in (k_pages, v_pages)]
    keep = (slots >= 0) & (slots < pages * page)
    for pool, rows in zip(want, (k, v)):
        pool[slots[keep] // page, slots[keep] % page] = rows[keep]
    cache = ncz.paged.Cache(k_pages, v_pages)
    ncz.paged.append(k, v, slots, cache)
    torch.cuda.synchronize()
    assert torch.equal(k_pages, want[0]) and torch.equal(v_pages, want[1])


@pytest.mark.parametrize("dim,kind", [(32, "plain"), (64, "odd"), (128, "interleaved")])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_quantises(ncz, dim, kind, dtype):
    """x / scale rounded to nearest even and saturated at 448, NaN kept: every
    finite 16-bit input pattern, bit for bit as torch rounds the clamped quotient."""
    kv, page = 3, 8
    bits = torch.arange(1 << 16, dtype=torch.int32, device="cuda").to(torch.int16).view(dtype)
    n = bits.numel() // (kv * dim) * (kv * dim)
    g = torch.Generator(device="cuda").manual_seed(1)
    k = bits[:n].view(-1, kv, dim)
    tokens = k.shape[0]
    v = torch.randn(tokens, kv, dim, generator=g, device="cuda").to(dtype)
    if kind == "odd":
        k, v = (torch.nn.functional.pad(x, (1, 0))[..., 1:] for x in (k, v))
    pages = -(-tokens // page)
    scales = torch.tensor([[1.0, 0.37, 3.0], [0.004, 1.0, 0.25]], device="cuda")
    for k_scale, v_scale in ((scales[0], scales[1]), (None, scales[1]), (None, None)):
        pools = [torch.zeros(pages, page, kv, dim, dtype=E4M3, device="cuda") for _ in range(2)]
        cache = ncz.paged.Cache(*pools, k_scale=k_scale, v_scale=v_scale)
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
        ncz.paged.append(k, v, slots, cache)
        torch.cuda.synchronize()
        for pool, rows, scale in zip(pools, (k, v), (k_scale, v_scale)):
            x = rows.float() / (1.0 if scale is None else scale[:, None])
            want = x.clamp(-448, 448).to(E4M3)
            got = pool.view(-1, kv, dim).view(torch.uint8)[slots].view(E4M3)
            nan = torch.isnan(x)
            assert torch.equal(torch.isnan(got.float()), nan)
            assert torch.equal(got.float()[~nan], want.float()[~nan])


def test_append_of_nothing(ncz):
    pool = pages_of(2, 4, 2, 32, F16, "plain")
    cache = ncz.paged.Cache(pool, pool.clone())
    empty = torch.zeros(0, 2, 32, dtype=F16, device="cuda")
    ncz.paged.append(empty, empty, torch.zeros(0, dtype=torch.int64, device="cuda"), cache)
    assert bool((pool == 3).all())


# ---------------------------------------------------------------- decode

def to_layout(x, layout):
    if layout == "heads_first":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "padded":
        wide = torch.zeros(*x.shape[:3], x.shape[3] + 16, device=x.device).to(x.dtype)
        wide[..., :x.shape[3]] = x.float()
        return wide[..., :x.shape[3]]
    return x


def run_decode(ncz, pr, out, *, window=0, layout="plain", k_scale=None, v_scale=None, q=None, o=None, lse=True, **kw):
    dev = {n: pr[n].cuda() for n in ("q", "k", "v", "table", "lens")}
    scales = [None if s is None else s.cuda() for s in (k_scale, v_scale)]
    cache = ncz.paged.Cache(to_layout(dev["k"], layout), to_layout(dev["v"], layout), k_scale=scales[0],
                            v_scale=scales[1])
    q = dev["q"] if q is None else q
    o = torch.full(pr["q"].shape, 7.0, dtype=out, device="cuda") if o is None else o
    lse = torch.full(pr["q"].shape[:2], 7.0, device="cuda") if lse else None
    ncz.paged.decode(q, cache, dev["table"], dev["lens"], o, scale=pr["scale"], window=window, lse=lse, **kw)
    torch.cuda.synchronize()
    return o.cpu(), None if lse is None else lse.cpu()


def check_decode(ncz, pr, out, *, window=0, k_scale=None, v_scale=None, **kw):
    want, want_lse, tol, tol_lse = P.decode_oracle(pr["q"], pr["k"], pr["v"], pr["table"], pr["lens"], pr["scale"],
                                                   window, k_scale, v_scale,
                                                   2.0 ** -11 if pr["k"].dtype == E4M3 and out == BF16 else 2.0 ** -17)
    o, lse = run_decode(ncz, pr, out, window=window, k_scale=k_scale, v_scale=v_scale, **kw)
    err = (o.double() - want).abs()
    assert bool(torch.isfinite(o).all())
    # the smallest step of a 16-bit output near zero: half a subnormal
    limit = tol + P.half_step(out) * (want.abs() + tol) + torch.finfo(out).smallest_normal * torch.finfo(out).eps
    assert bool((err <= limit).all()), float((err / limit).max())
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty)
    assert bool((o[empty] == 0).all())
    assert bool(((lse.double() - want_lse).abs()[~empty] <= tol_lse[~empty]).all())
    return o, lse


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 127, 128, 129, 255, 256, 257, 300]


@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [1, 3, 8, 12, 20])
def test_decode_short_lengths(ncz, dim, dtype, group):
    pr = P.decode_problem(len(LENS), 2 * group, 2, dim, 16, LENS, dtype, seed=dim + group)
    check_decode(ncz, pr, F32)
    check_decode(ncz, pr, dtype)
    # a table wide enough that rows might be long: even shares over the CTAs instead of clusters
    pr = P.decode_problem(len(LENS), 2 * group, 2, dim, 16, LENS, dtype, seed=dim + group, width=1500)
    check_decode(ncz, pr, F32)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [1, 7, 16, 33])
def test_decode_e4m3(ncz, dim, dtype, group):
    pr = P.decode_problem(len(LENS), 2 * group, 2, dim, 8, LENS, dtype, cache_dtype=E4M3, seed=dim + group)
    ks, vs = torch.tensor([0.05, 0.031]), torch.tensor([0.02, 1.3])
    check_decode(ncz, pr, F32, k_scale=ks, v_scale=vs)
    check_decode(ncz, pr, dtype, k_scale=ks)
    pr = P.decode_problem(len(LENS), 2 * group, 2, dim, 8, LENS, dtype, cache_dtype=E4M3, seed=dim + group, width=3000)
    check_decode(ncz, pr, dtype, k_scale=ks, v_scale=vs)


@pytest.mark.parametrize("page", [1, 2, 3, 7, 16, 30, 64, 257])
@pytest.mark.parametrize("layout", ["plain", "heads_first", "padded"])
def test_decode_page_sizes_and_layouts(ncz, page, layout):
    pr = P.decode_problem(5, 12, 3, 64, page, [200, 0, 77, 513, 1], BF16, seed=page)
    check_decode(ncz, pr, F32, layout=layout)


@pytest.mark.parametrize("batch,kv,lens", [(1, 1, [5000]), (1, 2, [9001]), (2, 1, [4096, 31]), (3, 5, [3000, 0, 2999])])
@pytest.mark.parametrize("dim,group,dtype,cache", [(128, 4, BF16, BF16), (64, 1, F16, F16), (16, 9, F16, F16),
                                                   (128, 32, BF16, BF16), (128, 8, BF16, E4M3), (32, 2, BF16, BF16)])
def test_decode_split_rows_are_joined(ncz, batch, kv, lens, dim, group, dtype, cache):
    pr = P.decode_problem(batch, kv * group, kv, dim, 16, lens, dtype, cache_dtype=cache, seed=kv + dim)
    ks = torch.full((kv,), 0.04) if cache == E4M3 else None
    check_decode(ncz, pr, F32, k_scale=ks)


@pytest.mark.parametrize("batch", [40, 700])
def test_decode_many_requests(ncz, batch):
    """More rows than CTAs, and more requests than a CTA has threads."""
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, 200 if batch > 100 else 900, batch).tolist()
    pr = P.decode_problem(batch, 4, 2, 32, 16, lens, F16, seed=batch)
    check_decode(ncz, pr, F32)


# Many query heads per K/V head: the tcgen05 kernel takes launches of at least
# two steps of 128 keys per SM (the table's width counts: a wide one is enough).
WIDE_LENS = [0, 1, 127, 128, 129, 900, 1000, 256, 385, 640, 17, 5]


def wide_problem(batch, group, kv, dim, page, lens, dtype, **kw):
    pr = P.decode_problem(batch, kv * group, kv, dim, page, lens, dtype, width=-(-(148 * 2 * 128) // page), **kw)
    return pr


@pytest.mark.parametrize("dim,group", [(64, 17), (64, 32), (64, 33), (64, 64), (64, 100), (64, 130), (128, 9), (128, 32),
                                       (128, 40), (128, 64), (128, 65), (128, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_many_heads_per_kv_head(ncz, dim, group, dtype):
    pr = wide_problem(len(WIDE_LENS), group, 1, dim, 16, WIDE_LENS, dtype, seed=dim + group)
    check_decode(ncz, pr, dtype)
    assert ncz.paged.sync_status() == 0


@pytest.mark.parametrize("dim,group,kv,page", [(64, 20, 3, 7), (128, 12, 2, 1), (128, 50, 2, 100), (64, 70, 1, 32)])
@pytest.mark.parametrize("layout", ["plain", "heads_first", "padded"])
def test_decode_many_heads_layouts_windows_and_items(ncz, dim, group, kv, page, layout):
    """Several items a CTA (60 requests), parts that end and begin inside CTAs, a
    window whose pages before it are gone, odd strides of q and o."""
    rng = np.random.default_rng(dim + group)
    lens = rng.integers(0, 900, 60).tolist()
    pr = wide_problem(60, group, kv, dim, page, lens, BF16, seed=page)
    check_decode(ncz, pr, BF16, layout=layout)
    for b, n in enumerate(lens):
        pr["table"][b, :max(0, n - 600) // page] = -1
    wide = torch.zeros(60, kv * group, dim + 3, dtype=BF16, device="cuda")
    wide[..., 1:dim + 1] = pr["q"].cuda()
    hold = torch.full((60, kv * group, dim + 5), 9.0, dtype=F16, device="cuda")
    o = hold[..., 3:dim + 3]
    check_decode(ncz, pr, F16, window=600, layout=layout, q=wide[..., 1:dim + 1], o=o)
    o.fill_(9.0)
    assert bool((hold == 9).all())
    assert ncz.paged.sync_status() == 0


def test_decode_many_heads_large_scores_and_absent_pages(ncz):
    pr = wide_problem(3, 24, 1, 128, 16, [1500, 2000, 900], F16, seed=8)
    ramp = torch.linspace(0.01, 8, 2000)
    for b in range(3):
        for j in range(int(pr["lens"][b])):
            p_, r = int(pr["table"][b, j // 16]), j % 16
            pr["k"][p_, r] *= ramp[j] if b != 1 else ramp[1999 - j]
    for scale in (1.0, -0.5, 0.0):
        pr["scale"] = scale
        check_decode(ncz, pr, F16)
    pr["table"][0, 20:60] = -1
    pr["table"][1, :] = 2**31 - 1
    pr["table"][2, 0] = pr["k"].shape[0]
    _, lse = check_decode(ncz, pr, F16)
    assert bool(torch.isinf(lse[1]).all())


def test_decode_many_heads_long_rows_match_few_heads(ncz):
    """20000 keys a request: every head's output is that of the same head decoded
    alone (warp MMAs), up to both roundings."""
    group, dim, n, page = 32, 128, 20000, 32
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(2 * n // page, page, 1, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(2, group, dim, generator=g, device="cuda").bfloat16()
    table = torch.randperm(2 * n // page, generator=g, device="cuda").int().view(2, -1)
    lens = i32([n, n - 77])
    cache = ncz.paged.Cache(k, v)
    o, one = torch.empty_like(q), torch.empty(2, 1, dim, device="cuda")
    ncz.paged.decode(q, cache, table, lens, o, scale=dim ** -0.5)
    for h in range(0, group, 5):
        ncz.paged.decode(q[:, h:h + 1], cache, table, lens, one, scale=dim ** -0.5)
        # P in 16 bits twice and f32 sums: 2^-9 of o, and 2^-16 of sum p |v| <= max |v| / 16 here
        limit = 2.0 ** -9 * one[:, 0].abs() + 2.0 ** -16 * float(v.float().abs().max())
        assert bool(((o[:, h].float() - one[:, 0]).abs() <= limit).all()), h
    assert ncz.paged.sync_status() == 0


def test_decode_wait_that_runs_out(ncz):
    """A step's scores that are never announced: the kernel stops by itself, the
    status word says so, and the next call is right again."""
    pr = wide_problem(4, 20, 1, 64, 16, [300, 400, 500, 600], F16, seed=1)
    lib = ncz.paged.lib()
    want, _ = run_decode(ncz, pr, F16)
    assert lib.ncz_paged_test_set_wait_limit(-1, 2_000_000) == 0  # about 1 ms
    assert lib.ncz_paged_test_drop_scores(-1, 1) == 0
    try:
        run_decode(ncz, pr, F16)
        with pytest.raises(ncz.FlashError, match="DeviceTimeout"):
            ncz.paged.sync_status()
    finally:
        assert lib.ncz_paged_test_drop_scores(-1, 0) == 0
        assert lib.ncz_paged_test_set_wait_limit(-1, 0) == 0
    got, _ = run_decode(ncz, pr, F16)
    assert ncz.paged.sync_status() == 0 and torch.equal(got, want)


@pytest.mark.parametrize("fill", [0x7F, 0xFF, 0x01, None])
@pytest.mark.parametrize("lens", [[300, 400, 500, 600], [9000]])
def test_decode_wait_that_runs_out_on_any_workspace(ncz, lens, fill):
    """A launch that stops early leaves records of shared rows unwritten: whatever
    the workspace held there, nothing outside o and lse is touched."""
    pr = wide_problem(len(lens), 20, 2, 64, 16, lens, F16, seed=3)
    dev = {n: pr[n].cuda() for n in ("q", "k", "v", "table", "lens")}
    cache = ncz.paged.Cache(dev["k"], dev["v"])
    lib = ncz.paged.lib()
    workspace = ncz.paged.decode_workspace(cache, 40)
    if fill is None:
        workspace.random_(0, 256, generator=torch.Generator(device="cuda").manual_seed(5))
    else:
        workspace.fill_(fill)
    n = pr["q"].numel()
    around = torch.full((n + 8192,), 3.0, dtype=F16, device="cuda")
    o = around[4096:4096 + n].view(pr["q"].shape)
    assert lib.ncz_paged_test_set_wait_limit(-1, 2_000_000) == 0  # about 1 ms
    assert lib.ncz_paged_test_drop_scores(-1, 1) == 0
    try:
        ncz.paged.decode(dev["q"], cache, dev["table"], dev["lens"], o, scale=pr["scale"], workspace=workspace)
        with pytest.raises(ncz.FlashError, match="DeviceTimeout"):
            ncz.paged.sync_status()
    finally:
        assert lib.ncz_paged_test_drop_scores(-1, 0) == 0
        assert lib.ncz_paged_test_set_wait_limit(-1, 0) == 0
    assert bool((around[:4096] == 3).all()) and bool((around[4096 + n:] == 3).all())
    got, _ = run_decode(ncz, pr, F16, workspace=workspace)
    want, _ = run_decode(ncz, pr, F16)
    assert ncz.paged.sync_status() == 0 and torch.equal(got, want)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 100, 1000])
def test_decode_window(ncz, window):
    """The pages before a window are given back (-1): nothing of them is read."""
    lens = [0, 1, 50, 300, 301, 999, 1000, 1001]
    page = 7
    pr = P.decode_problem(len(lens), 6, 3, 64, page, lens, F16, seed=window)
    check_decode(ncz, pr, F32, window=window)
    for b, n in enumerate(lens):
        pr["table"][b, :max(0, n - window) // page] = -1
    check_decode(ncz, pr, F16, window=window)


def test_decode_absent_pages_and_bad_ids(ncz):
    """Ids outside the cache leave their keys out, in the middle too; a row of
    none of them left is empty."""
    pr = P.decode_problem(4, 8, 2, 128, 16, [500, 90, 33, 700], BF16, seed=3)
    pr["table"][0, 3:9] = -1
    pr["table"][0, 20] = 2**31 - 1
    pr["table"][1, :] = pr["k"].shape[0]
    pr["table"][3, :20] = -2**31
    o, lse = check_decode(ncz, pr, F32)
    assert bool(torch.isinf(lse[1]).all()) and bool((o[1] == 0).all())


def test_decode_lengths_past_the_table_are_clamped(ncz):
    pr = P.decode_problem(3, 4, 2, 64, 16, [64, 30, 48], F16, width=4)
    pr["lens"] = torch.tensor([2**31 - 1, -5, 48], dtype=torch.int32)
    check_decode(ncz, pr, F32)


def test_decode_table_of_no_columns(ncz):
    pr = P.decode_problem(2, 4, 2, 64, 16, [0, 0], F16)
    pr["table"] = torch.zeros(2, 0, dtype=torch.int32)
    pr["lens"] = torch.tensor([9, 0], dtype=torch.int32)
    o, lse = run_decode(ncz, pr, F32)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("fill", [math.inf, -math.inf, -65504.0, float("nan")])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_ignores_what_lies_outside(ncz, fill, dtype):
    pr = P.decode_problem(6, 4, 4, 64, 16, [1, 17, 40, 130, 300, 5], dtype, fill=fill, seed=5)
    check_decode(ncz, pr, F32)


def test_decode_large_scores(ncz):
    """Scores of several hundred, rising and falling along the keys: the running
    maximum moves, and P spans its whole range."""
    pr = P.decode_problem(3, 8, 2, 64, 16, [700, 1000, 900], F16, seed=8)
    ramp = torch.linspace(0.01, 12, 1000)
    for b in range(3):
        for j in range(int(pr["lens"][b])):
            p_, r = int(pr["table"][b, j // 16]), j % 16
            pr["k"][p_, r] *= ramp[j] if b != 1 else ramp[999 - j]
    pr["scale"] = 1.0
    check_decode(ncz, pr, F32)
    pr["scale"] = -0.5
    check_decode(ncz, pr, F32)
    pr["scale"] = 0.0
    check_decode(ncz, pr, F32)


def test_decode_heavy_tail(ncz):
    """One key far above thousands of others whose weights are each 2^-25: their
    sum is kept."""
    n = 6000
    pr = P.decode_problem(1, 2, 1, 64, 16, [n], F16, seed=9)
    pr["q"].zero_()
    pr["q"][..., 0] = 1.0
    pr["k"][...] = 0
    page0 = int(pr["table"][0, 0])
    pr["k"][page0, 3, :, 0] = 25 * math.log(2)
    pr["v"][...] = 1.0
    pr["v"][page0, 3] = 0.0
    pr["scale"] = 1.0
    o, _ = run_decode(ncz, pr, F32)
    weight = (n - 1) * math.exp(-float(pr["k"][page0, 3, 0, 0]))
    want = weight / (1 + weight)
    assert float((o - want).abs().max()) <= want * 1e-3  # f16's subnormals would lose all of it


def test_decode_nonfinite_inputs_stay_in_their_rows(ncz):
    pr = P.decode_problem(3, 4, 2, 64, 16, [100, 200, 300], F16, seed=4)
    pr["q"][1, 2, 5] = float("nan")
    pr["v"][int(pr["table"][2, 4]), 3, 0, 7] = float("nan")
    o, lse = run_decode(ncz, pr, F32)
    assert bool(torch.isnan(o[1, 2]).all()) and bool(torch.isnan(lse[1, 2]))
    assert bool(torch.isnan(o[2, :2, 7]).all())
    bad = torch.isnan(o)
    bad[1, 2] = False
    bad[2, :2, 7] = False
    assert not bool(bad.any()) and int(torch.isnan(lse).sum()) == 1


def test_decode_bf16_queries_outside_f16_range(ncz):
    """bf16 q against an e4m3 cache: magnitudes no f16 holds."""
    pr = P.decode_problem(4, 4, 2, 64, 16, [50, 60, 70, 80], BF16, cache_dtype=E4M3, seed=6)
    pr["q"][0] *= 2.0 ** 40
    pr["q"][1] *= 2.0 ** -60
    pr["q"][2, 0] = 0
    ks = torch.tensor([2.0 ** -6, 2.0 ** -6])
    for b, scale in ((0, 2.0 ** -44), (1, 2.0 ** 57), (2, 0.125), (3, 0.125)):
        one = dict(pr, q=pr["q"][b:b + 1], table=pr["table"][b:b + 1], lens=pr["lens"][b:b + 1], scale=scale)
        check_decode(ncz, one, F32, k_scale=ks)


@pytest.mark.parametrize("kind", ["odd", "transposed", "broadcast"])
@pytest.mark.parametrize("out", [F32, BF16])
def test_decode_strides_of_q_and_o(ncz, kind, out):
    batch, heads, dim = 4, 6, 64
    pr = P.decode_problem(batch, heads, 3, dim, 16, [30, 300, 0, 129], BF16, seed=2)
    if kind == "broadcast":
        pr["q"] = pr["q"][:, :1].expand(batch, heads, dim).contiguous()
    q = pr["q"].cuda()
    if kind == "odd":
        wide = torch.zeros(batch, heads, dim + 3, dtype=BF16, device="cuda")
        wide[..., 1:dim + 1] = q
        q = wide[..., 1:dim + 1]
        hold = torch.full((batch, heads, dim + 5), 9.0, dtype=out, device="cuda")
        o = hold[..., 3:dim + 3]
    elif kind == "transposed":
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
        hold = torch.full((heads, batch, dim), 9.0, dtype=out, device="cuda")
        o = hold.transpose(0, 1)
    else:
        q = q[:, :1].expand(batch, heads, dim)
        hold = torch.full((batch + 2, heads, dim), 9.0, dtype=out, device="cuda")
        o = hold[1:batch + 1]
    check_decode(ncz, pr, out, q=q, o=o)
    o.fill_(9.0)
    assert bool((hold == 9).all())  # nothing beside the rows was written


def test_decode_without_lse_and_repeatable(ncz):
    pr = P.decode_problem(9, 16, 4, 128, 16, [1000, 3, 555, 0, 64, 128, 2000, 77, 1], BF16, seed=12)
    a, _ = run_decode(ncz, pr, BF16, lse=False)
    b, _ = run_decode(ncz, pr, BF16)
    c, _ = run_decode(ncz, pr, BF16)
    assert torch.equal(a, b) and torch.equal(b, c)


def test_decode_offsets_past_32_bits(ncz):
    """A cache of more than 2^32 bytes per pool (and 2^31 elements), pages at its far end."""
    dim, kv, page = 128, 8, 16
    pages = (2**31 // (dim * kv * page)) + 70
    k_pages = torch.empty(pages, page, kv, dim, dtype=F16, device="cuda")
    v_pages = torch.empty_like(k_pages)
    ids = [pages - 1, 0, pages - 3, 7, pages - 69]
    small = P.decode_problem(1, kv, kv, dim, page, [75], F16, seed=1)
    order = [int(x) for x in small["table"][0, :5]]
    cache = ncz.paged.Cache(k_pages, v_pages)
    slots = torch.tensor([ids[j // page] * page + j % page for j in range(75)], device="cuda")
    at = [(order[j // page], j % page) for j in range(75)]
    k, v = (torch.stack([small[n][p, r] for p, r in at]).cuda() for n in ("k", "v"))
    ncz.paged.append(k, v, slots, cache)
    o = torch.empty(1, kv, dim, device="cuda")
    ncz.paged.decode(small["q"].cuda(), cache, i32([ids]), i32([75]), o, scale=small["scale"])
    want, _, tol, _ = P.decode_oracle(small["q"], small["k"], small["v"], small["table"], small["lens"], small["scale"])
    assert bool(((o.cpu().double() - want).abs() <= tol + 2.0 ** -24).all())


@pytest.mark.parametrize("lens,dim", [([900, 3, 1000, 0, 64], 64), ([9000, 1], 128)])
def test_decode_workspace_of_any_contents(ncz, lens, dim):
    """One workspace for calls in a row, whatever it held before: ones, random
    bytes, the parts and flags of other shapes; and a captured call replayed on it."""
    pr = P.decode_problem(len(lens), 8, 2, dim, 16, lens, BF16, seed=dim)
    other = P.decode_problem(3, 8, 2, dim, 16, [500, 77, 1200], BF16, seed=2)
    want, want_lse = run_decode(ncz, pr, F32)
    dev = {n: pr[n].cuda() for n in ("q", "k", "v", "table", "lens")}
    cache = ncz.paged.Cache(dev["k"], dev["v"])
    workspace = ncz.paged.decode_workspace(cache, 8)
    g = torch.Generator(device="cuda").manual_seed(1)
    o, lse = torch.zeros(pr["q"].shape, device="cuda"), torch.zeros(pr["q"].shape[:2], device="cuda")

    def call():
        ncz.paged.decode(dev["q"], cache, dev["table"], dev["lens"], o, scale=pr["scale"], lse=lse, workspace=workspace)

    for fill in (0xFF, 0, None):
        if fill is None:
            workspace.random_(0, 256, generator=g)
        else:
            workspace.fill_(fill)
        for _ in range(3):
            o.fill_(5.0)
            call()
            assert torch.equal(o.cpu(), want) and torch.equal(lse.cpu(), want_lse)
            run_decode(ncz, other, F32, workspace=workspace)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(20):
        o.fill_(5.0)
        graph.replay()
        assert torch.equal(o.cpu(), want)
        run_decode(ncz, other, F32, workspace=workspace)


# ---------------------------------------------------------------- streams, graphs, refusals

def test_calls_on_another_stream(ncz):
    pr = P.decode_problem(4, 8, 2, 128, 16, [1000, 3000, 64, 0], BF16, seed=21)
    want, _ = run_decode(ncz, pr, BF16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream):
        got, _ = run_decode(ncz, pr, BF16, stream=stream)
        assert torch.equal(got, want)
    with torch.cuda.stream(side):
        got, _ = run_decode(ncz, pr, BF16)
    assert torch.equal(got, want)


def test_calls_at_once_on_several_streams(ncz):
    """Every form of decode (clusters for few rows, even shares with a join, tcgen05),
    plan and append side by side, eager, each with its own workspace."""
    problems = [P.decode_problem(2, 8, 2, 128, 16, [900, 31], BF16, seed=1),
                P.decode_problem(3, 8, 8, 64, 16, [9000, 1, 2500], BF16, seed=2),
                wide_problem(3, 32, 1, 128, 16, [5000, 0, 7000], BF16, seed=3),
                wide_problem(2, 20, 2, 64, 16, [6000, 100], BF16, seed=4)]
    wants = [run_decode(ncz, pr, BF16)[0] for pr in problems]
    runs = []
    for pr in problems:
        dev = {n: pr[n].cuda() for n in ("q", "k", "v", "table", "lens")}
        cache = ncz.paged.Cache(dev["k"], dev["v"])
        runs.append((torch.cuda.Stream(), dev, cache, ncz.paged.decode_workspace(cache, pr["q"].shape[1]),
                     [torch.zeros(pr["q"].shape, dtype=BF16, device="cuda") for _ in range(8)]))
    held, added = i32(4 * (np.arange(500) % 9)), i32(np.arange(500) % 5)  # whole pages held: all slots differ
    free = i32(np.arange(3000)[::-1].copy())
    plans = [(torch.cuda.Stream(), torch.full((500, 16), 9, dtype=torch.int32, device="cuda"), i32([3000]),
              torch.zeros(500, dtype=torch.int32, device="cuda"),
              torch.zeros(1200, dtype=torch.int64, device="cuda")) for _ in range(2)]
    rows = torch.randn(1200, 2, 64, dtype=BF16, device="cuda")
    pools = [[torch.zeros(3000, 4, 2, 64, dtype=BF16, device="cuda") for _ in range(2)] for _ in plans]
    targets = [ncz.paged.Cache(*pool) for pool in pools]
    torch.cuda.synchronize()
    for i in range(8):
        for (stream, dev, cache, workspace, outs), pr in zip(runs, problems):
            ncz.paged.decode(dev["q"], cache, dev["table"], dev["lens"], outs[i], scale=pr["scale"],
                             workspace=workspace, stream=stream)
        for (stream, table, count, lens, slots), target in zip(plans, targets):
            if i == 0:
                ncz.paged.plan(held, added, free, count, table, lens, slots, page_size=4, stream=stream)
            ncz.paged.append(rows, rows, slots, target, stream=stream)
    torch.cuda.synchronize()
    assert ncz.paged.sync_status() == 0
    for (_, _, _, _, outs), want in zip(runs, wants):
        assert all(torch.equal(o.cpu(), want) for o in outs)
    slots = plans[0][4]
    assert int((slots >= 0).sum()) == int(added.sum()) and torch.equal(slots, plans[1][4])
    for pool in pools:
        for x in pool:
            assert torch.equal(x.view(-1, 2, 64)[slots[slots >= 0]], rows[:int(added.sum())])


def test_two_graphs_replayed_side_by_side(ncz):
    """Graphs captured without a workspace of their own hold one each."""
    problems = [P.decode_problem(1, 8, 1, 128, 16, [n], BF16, seed=n) for n in (9000, 7001)]
    wants = [run_decode(ncz, pr, BF16)[0] for pr in problems]
    graphs, outs, keep = [], [], []
    for pr in problems:
        dev = {n: pr[n].cuda() for n in ("q", "k", "v", "table", "lens")}
        cache = ncz.paged.Cache(dev["k"], dev["v"])
        o = torch.zeros(pr["q"].shape, dtype=BF16, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ncz.paged.decode(dev["q"], cache, dev["table"], dev["lens"], o, scale=pr["scale"])
        graphs.append(graph)
        outs.append(o)
        keep.append((dev, cache))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for o, want in zip(outs, wants):
        assert torch.equal(o.cpu(), want)


def test_wrapper_refusals(ncz):
    pr = P.decode_problem(2, 4, 2, 64, 16, [5, 6], F16)
    d = {n: pr[n].cuda() for n in ("q", "k", "v", "table", "lens")}
    k, v = torch.zeros_like(d["k"]), torch.zeros_like(d["v"])
    cache = ncz.paged.Cache(k, v)
    o = torch.zeros_like(d["q"])
    bad = pytest.raises(ncz.FlashError)
    for args in ((k, v[:1]), (k, v.bfloat16()), (k.float(), v.float()), (k[..., ::2], v[..., ::2]),
                 (k[..., 1:33], v[..., 1:33]), (k.expand(4, *k.shape)[:, 0], v), (k[:, :, :, :48], v[:, :, :, :48])):
        with bad:
            ncz.paged.Cache(*args)
    with bad:
        ncz.paged.Cache(k, v, k_scale=torch.ones(2, device="cuda"))  # not an 8-bit cache
    with bad:
        ncz.paged.Cache(k.to(E4M3), v.to(E4M3), k_scale=torch.ones(1, device="cuda"))
    good = dict(scale=0.125)
    for q_, t_, l_, o_, kw in (
            (d["q"].bfloat16(), d["table"], d["lens"], o, good), (d["q"][:, :3], d["table"], d["lens"], o[:, :3], good),
            (d["q"], d["table"].long(), d["lens"], o, good), (d["q"], d["table"], d["lens"].long(), o, good),
            (d["q"], d["table"][:1], d["lens"], o, good), (d["q"], d["table"], d["lens"][:1], o, good),
            (d["q"], d["table"], d["lens"], o[:1], good), (d["q"], d["table"], d["lens"], o.double(), good),
            (d["q"].cpu(), d["table"], d["lens"], o, good), (d["q"], d["table"], d["lens"], o, dict(scale=1.0, window=-1)),
            (d["q"], d["table"], d["lens"], o[:, :1].expand_as(o), good),
            (d["q"], d["table"], d["lens"], o, dict(scale=1.0, lse=torch.zeros(2, 3, device="cuda"))),
            (d["q"], d["table"], d["lens"], o, dict(scale=1.0, workspace=torch.zeros(64, device="cuda")))):
        with bad:
            ncz.paged.decode(q_, cache, t_, l_, o_, **kw)
    slots = torch.zeros(2, dtype=torch.int64, device="cuda")
    rows = torch.zeros(2, 2, 64, dtype=F16, device="cuda")
    for k_, v_, s_ in ((rows, rows[:1], slots), (rows.bfloat16(), rows.bfloat16(), slots), (rows, rows, slots[:1]),
                       (rows, rows, slots.int()), (rows[:, :1], rows[:, :1], slots), (rows.cpu(), rows.cpu(), slots)):
        with bad:
            ncz.paged.append(k_, v_, s_, cache)
    ints = i32([1, 2])
    with bad:
        ncz.paged.plan(ints, ints[:1], ints, ints[:1], d["table"], ints.clone(), slots, page_size=16)
    with bad:
        ncz.paged.plan(ints, ints, ints, ints[:1], d["table"], ints.clone(), slots, page_size=0)
    with bad:
        ncz.paged.plan(ints, ints, ints, ints[:1], d["table"], ints.clone(), slots.int(), page_size=16)
    torch.cuda.synchronize()
    assert bool((o == 0).all()) and bool((k == 0).all())


# ---------------------------------------------------------------- together

def test_generate_after_the_forward(ncz):
    """A prompt through the forward (`launch`), its K/V into pages, then token by
    token through plan, append and decode inside one captured graph: every step's
    output is the last row of the forward over the whole sequence."""
    heads, dim, page, pages = 4, 64, 16, 64
    prompts, steps = [37, 1, 130], 20
    n = len(prompts)
    total = max(prompts) + steps
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = [(torch.randn(n, heads, total, dim, generator=g, device="cuda") * 0.7).half() for _ in range(3)]
    scale = dim ** -0.5

    def forward(b, length):  # the whole sequence of request b through the framework's forward, causal
        q, k, v = (x[b, :, :length].contiguous() for x in qkv)
        o = torch.zeros(heads, length, dim, device="cuda")
        st = length * dim
        ncz.launch(q.view(-1), k.view(-1), v.view(-1), o.view(-1),
                   ncz.Options(seq_len=length, head_dim=dim, q_stride=st, k_stride=st, v_stride=st, o_stride=st,
                               scale=scale, batch_heads=heads, causal=True))
        return o

    pool = [torch.full((pages, page, heads, dim), float("nan"), dtype=F16, device="cuda") for _ in range(2)]
    cache = ncz.paged.Cache(*pool)
    lens, added = i32([0] * n), i32(prompts)
    free, count = i32(np.arange(pages)), i32([pages])
    table = torch.full((n, 16), -1, dtype=torch.int32, device="cuda")
    slots = torch.empty(sum(prompts), dtype=torch.int64, device="cuda")
    ncz.paged.plan(lens, added, free, count, table, lens, slots, page_size=page)
    rows = [torch.cat([x[b, :, :m].transpose(0, 1) for b, m in enumerate(prompts)]) for x in qkv[1:]]
    ncz.paged.append(rows[0], rows[1], slots, cache)

    one = i32([1] * n)
    step_slots = torch.empty(n, dtype=torch.int64, device="cuda")
    q_now, k_now, v_now = (torch.zeros(n, heads, dim, dtype=F16, device="cuda") for _ in range(3))
    o = torch.zeros(n, heads, dim, device="cuda")
    workspace = ncz.paged.decode_workspace(cache, heads)

    def step():
        ncz.paged.plan(lens, one, free, count, table, lens, step_slots, page_size=page)
        ncz.paged.append(k_now, v_now, step_slots, cache)
        ncz.paged.decode(q_now, cache, table, lens, o, scale=scale, workspace=workspace)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # captured, not run: lengths and pages stay as they are
        step()
    for i in range(steps):
        for b, m in enumerate(prompts):
            for to, x in zip((q_now, k_now, v_now), qkv):
                to[b] = x[b, :, m + i]
        graph.replay()
        for b, m in enumerate(prompts):
            want = forward(b, m + i + 1)[:, -1]
            # the forward rounds P to f16 (2^-11 of sum p |v| <= max |v|, twice: P and its sum)
            limit = 2 * 2.0 ** -11 * float(qkv[2][b].abs().max())
            assert float((o[b] - want).abs().max()) <= limit, (i, b)
    assert lens.tolist() == [m + steps for m in prompts]
    used = sum(-(-(m + steps) // page) for m in prompts)
    assert count.tolist() == [pages - used]
    assert ncz.sync_status() == 0


def test_compare_paged_record(ncz):
    import importlib

    compare = importlib.import_module("not-cute-zig_b200.compare")
    for cache in ("f16", "bf16", "e4m3"):
        rec = compare.compare_paged(ncz, 3, 8, 2, 64, 333, cache)
        assert rec["correct"] and rec["kernel"] == "paged_decode", rec
