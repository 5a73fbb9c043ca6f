"""Edges of the paged-cache operators on the GPU that tests/test_paged_gpu.py leaves
out: calls on a device that is busy, scales and values at the ends of their types, and
the rounding of P, each against the oracles of tests/paged_cases.py or a bound derived
beside it."""
import numpy as np
import pytest

from tests import paged_cases as P
from tests import paged_edge_cases as E

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

F32, F16, BF16, E4M3 = P.F32, P.F16, P.BF16, P.E4M3


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- plan

@pytest.mark.parametrize("n", [1, 300, 9000])
def test_plan_while_other_kernels_hold_the_sms(ncz, n):
    """Clusters that start when SMs fall free, their CTAs not at the same time: every call's
    slots, lengths, counts and table are the oracle's."""
    page, calls = 16, 24
    rng = np.random.default_rng(n)
    held = rng.integers(0, 40, n).astype(np.int32)
    added = rng.integers(0, 5, n).astype(np.int32)
    width = 4
    have = -(-held // page)
    need = -(-(held + added) // page) - have
    ids = rng.permutation(int(have.sum() + need.sum()) + 5).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    table[np.arange(width)[None, :] < have[:, None]] = ids[:have.sum()]
    free = ids[have.sum():]
    capacity = int(added.sum()) + 3
    want = P.plan_oracle(held, added, free, len(free), table, page, capacity)
    given = [i32(x) for x in (held, added, free, [len(free)])]
    outs = []
    for _ in range(calls):
        made = lambda k, dt=torch.int32: torch.full((k,), -77, dtype=dt, device="cuda")  # noqa: E731
        outs.append({"block_table": i32(table), "seq_lens": made(n), "slots": made(capacity, torch.int64),
                     "positions": made(capacity), "starts": made(n + 1), "left": made(1), "status": made(4)})
    x = torch.randn(2048, 2048, device="cuda", dtype=BF16)
    streams = [torch.cuda.Stream() for _ in range(4)]
    busy = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        with torch.cuda.stream(busy):
            for _ in range(4):
                x @ x
        ncz.paged.plan(*given, o["block_table"], o["seq_lens"], o["slots"], page_size=page, positions=o["positions"],
                       starts=o["starts"], left=o["left"], status=o["status"], stream=streams[i % 4])
    torch.cuda.synchronize()
    for o in outs:
        for name, value in want.items():
            assert np.array_equal(o[name].cpu().numpy(), value), name


# ---------------------------------------------------------------- decode, many query heads per K/V head

@pytest.mark.parametrize("dim,group", [(64, 20), (128, 20), (64, 40), (128, 64), (64, 100), (128, 128)])
@pytest.mark.parametrize("lens", [[300, 400, 500, 600], [9000]])
def test_decode_stops_when_one_softmax_warp_gives_up_at_the_merge(ncz, dim, group, lens):
    """One of the four warps that merge an item leaves just before: the others must not wait for
    it.  The launch ends, the status word says so, and the next call is right again."""
    pr = P.decode_problem(len(lens), group, 1, dim, 16, lens, F16, width=-(-(148 * 2 * 128) // 16), seed=dim + group)
    dev = {n: pr[n].cuda() for n in ("q", "k", "v", "table", "lens")}
    cache = ncz.paged.Cache(dev["k"], dev["v"])
    outs = [torch.zeros(pr["q"].shape, dtype=F16, device="cuda") for _ in range(3)]
    lib = ncz.paged.lib()

    def call(o):
        ncz.paged.decode(dev["q"], cache, dev["table"], dev["lens"], o, scale=pr["scale"])

    call(outs[0])
    assert ncz.paged.sync_status() == 0
    assert lib.ncz_paged_test_set_wait_limit(-1, 2_000_000) == 0  # about 1 ms
    assert lib.ncz_paged_test_leave_merge(-1, 1) == 0
    try:
        call(outs[1])
        with pytest.raises(ncz.FlashError, match="DeviceTimeout"):
            ncz.paged.sync_status()
    finally:
        assert lib.ncz_paged_test_leave_merge(-1, 0) == 0
        assert lib.ncz_paged_test_set_wait_limit(-1, 0) == 0
    call(outs[2])
    assert ncz.paged.sync_status() == 0 and torch.equal(outs[0], outs[2])


# ---------------------------------------------------------------- decode, scales and values at the ends of their types

@pytest.mark.parametrize("dim,group,width,out", [(64, 2, 40, F32), (128, 4, 2400, BF16), (64, 20, 2400, BF16),
                                                 (128, 40, 2400, BF16), (32, 20, 40, BF16)])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-45])
def test_decode_of_large_bf16_scores_at_scale_zero(ncz, dim, group, width, out, scale):
    """Scores of 1e36 times 0 are 0: every key weighs the same, o is the mean of V and lse = ln n.
    (1e-45, the smallest f32, times log2 e stays the smallest f32: scores of 1e-9, below f32's
    step at a weight of 1.)  Bounds: weights are exact, V's sum of n terms is off by at most
    n 2^-23 of sum |v|, o by a rounding; log2 of up to 300 by 2^-20 (f32's step at 8), lse by 2^-22 more."""
    lens = [1, 300, 129, 0, 17]
    pr = P.decode_problem(5, 2 * group, 2, dim, 16, lens, BF16, seed=dim + group, width=width)
    pr["q"] *= 1e18
    pr["k"] = torch.where(torch.isnan(pr["k"]), pr["k"], pr["k"] * 1e17)
    dev = {n: pr[n].cuda() for n in ("q", "k", "v", "table", "lens")}
    o = torch.full(pr["q"].shape, 7.0, dtype=out, device="cuda")
    lse = torch.full(pr["q"].shape[:2], 7.0, device="cuda")
    ncz.paged.decode(dev["q"], ncz.paged.Cache(dev["k"], dev["v"]), dev["table"], dev["lens"], o, scale=scale, lse=lse)
    for b, n in enumerate(lens):
        if n == 0:
            assert bool((o[b] == 0).all()) and bool((lse[b] == -torch.inf).all())
            continue
        rows = torch.cat([pr["v"][int(pr["table"][b, j])] for j in range(-(-n // 16))])[:n].double()
        mean, size = rows.mean(0), rows.abs().mean(0)
        want = mean.repeat_interleave(group, 0)
        limit = ((n + 4) * 2.0 ** -23 * size + P.half_step(out) * (mean.abs() + size * 2.0 ** -12)).repeat_interleave(group, 0)
        assert bool(((o[b].cpu().double() - want).abs() <= limit).all()), b
        assert float((lse[b].cpu().double() - np.log(n)).abs().max()) <= 2.0 ** -19, b


@pytest.mark.parametrize("dim,group,width", [(64, 2, 40), (64, 20, 2400), (128, 40, 2400)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_scale_zero_keeps_nan_and_infinity(ncz, dim, group, width, dtype):
    """0 times an infinite or NaN score is NaN, in the rows of that query or key alone."""
    pr = P.decode_problem(3, 2 * group, 2, dim, 16, [40, 50, 60], dtype, seed=dim, width=width)
    pr["q"][0, 0, 3] = float("inf")
    pr["q"][1, 1, 0] = float("nan")
    pr["k"][int(pr["table"][2, 1]), 5, 1, 7] = float("inf")
    dev = {n: pr[n].cuda() for n in ("q", "k", "v", "table", "lens")}
    o = torch.zeros(pr["q"].shape, dtype=dtype, device="cuda")
    ncz.paged.decode(dev["q"], ncz.paged.Cache(dev["k"], dev["v"]), dev["table"], dev["lens"], o, scale=0.0)
    bad = torch.isnan(o).all(-1)
    want = torch.zeros_like(bad)
    want[0, 0] = want[1, 1] = True
    want[2, group:] = True
    assert torch.equal(torch.isnan(o).any(-1), bad) and torch.equal(bad, want)


@pytest.mark.parametrize("dim,group", [(32, 3), (64, 16), (128, 8)])
@pytest.mark.parametrize("top", [127, -133])
def test_decode_bf16_queries_at_the_ends_of_their_range_over_e4m3(ncz, dim, group, top):
    """Rows of q whose largest element is 1.5 2^127, or the smallest bf16 there is, against an
    8-bit cache: as the definition says, not infinity or 0.  Scores as in decode_oracle."""
    lens = [70, 3, 200]
    pr = P.decode_problem(3, 2 * group, 2, dim, 16, lens, BF16, cache_dtype=E4M3, seed=dim + group, fill=0.0)
    pr["k"] = (pr["k"].float() / 384).to(E4M3)
    g = torch.Generator().manual_seed(top + 200)
    sign = torch.where(torch.rand(pr["q"].shape, generator=g) < 0.5, -1.0, 1.0)
    if top > 0:
        q = sign.double() * 1.5 * 2.0 ** 127 * (torch.rand(pr["q"].shape, generator=g) < 0.5)
    else:
        q = sign.double() * 2.0 ** -133
    pr["q"] = q.to(BF16)
    k_scale = torch.tensor([1.0, 0.5]) if top > 0 else torch.tensor([2.0 ** 60, 2.0 ** 61])
    pr["scale"] = 2.0 ** -125 if top > 0 else 2.0 ** 75
    want, want_lse, tol, tol_lse = P.decode_oracle(pr["q"], pr["k"], pr["v"], pr["table"], pr["lens"], pr["scale"],
                                                   0, k_scale)
    dev = {n: pr[n].cuda() for n in ("q", "k", "v", "table", "lens")}
    o, lse = torch.zeros(pr["q"].shape, device="cuda"), torch.zeros(pr["q"].shape[:2], device="cuda")
    ncz.paged.decode(dev["q"], ncz.paged.Cache(dev["k"], dev["v"], k_scale=k_scale.cuda()), dev["table"], dev["lens"], o,
                     scale=pr["scale"], lse=lse)
    assert bool(((o.cpu().double() - want).abs() <= tol + P.half_step(F32) * want.abs()).all())
    assert bool(((lse.cpu().double() - want_lse).abs() <= tol_lse).all())


# ---------------------------------------------------------------- decode, the rounding of P

KINDS = [(F16, F16, F32), (F16, F16, F16), (BF16, BF16, F32), (BF16, BF16, BF16), (BF16, E4M3, BF16), (BF16, E4M3, F32),
         (F16, E4M3, F16), (F16, E4M3, F32)]


@pytest.mark.parametrize("dim,group,width", [(32, 1, 1), (64, 8, 40), (128, 12, 40), (128, 20, 2400)])
@pytest.mark.parametrize("q_dtype,dtype", [(F16, F16), (BF16, BF16), (BF16, E4M3), (F16, E4M3)])
def test_decode_one_weight_in_f32(ncz, dim, group, width, q_dtype, dtype):
    """f32 o holds a weight to f32's bits: P goes to the tensor cores in as many parts as that takes."""
    b = E.two_keys(dtype)
    n, page = len(b), 16
    k, v = (torch.zeros(n, page, 1, dim) for _ in range(2))
    k[:, 1, 0, 0] = b
    v[:, 1] = 1.0
    q = torch.zeros(n, group, dim, dtype=q_dtype, device="cuda")
    q[..., 0] = 1.0
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(n)
    o, lse = torch.zeros(n, group, dim, device="cuda"), torch.zeros(n, group, device="cuda")
    cache = ncz.paged.Cache(k.to(dtype).cuda(), v.to(dtype).cuda())
    ncz.paged.decode(q, cache, table, i32([2] * n), o, scale=1.0, lse=lse)
    w = torch.exp(b.double())[:, None, None]
    kind, count = E.parts_of(dtype, F32)
    limit = E.TWO_KEYS_BOUND + E.weight_error(kind, count)[0]
    assert float(((o.cpu().double() - w / (1 + w)).abs() / (w / (1 + w))).max()) <= limit
    # ln of the sum: 5.25 2^-22 of it as above, log2 (2^-23) and a rounding of up to 0.7
    assert float((lse.cpu().double() - torch.log1p(w[..., 0])).abs().max()) <= 7 * 2.0 ** -22


@pytest.mark.parametrize("down", [10.3, 21.7, 25.3, 29.6, 33.0, 36.5])
@pytest.mark.parametrize("n,group,width", [(3000, 2, 0), (700, 20, 2400), (700, 3, 0), (700, 70, 2400)])
@pytest.mark.parametrize("q_dtype,dtype,out", KINDS)
def test_decode_sum_of_small_weights(ncz, n, group, width, q_dtype, dtype, out, down):
    """Thousands of keys far below one: their sum is kept to the rounding of P's parts, which for
    f16 parts has an absolute term of 2^-33 of the largest weight a key."""
    dim, page = 64, 16
    pages = -(-n // page)
    k, v = torch.zeros(pages, page, 1, dim), torch.ones(pages, page, 1, dim)
    scale = down * float(np.log(2))
    k[pages // 2, 3, :, 0] = 1.0
    v[pages // 2, 3] = 0.0
    q = torch.zeros(1, group, dim, dtype=q_dtype, device="cuda")
    q[..., 0] = 1.0
    table = torch.full((1, max(width, pages)), -1, dtype=torch.int32, device="cuda")
    table[0, :pages] = torch.arange(pages)
    o = torch.zeros(1, group, dim, dtype=out, device="cuda")
    cache = ncz.paged.Cache(k.to(dtype).cuda(), v.to(dtype).cuda())
    ncz.paged.decode(q, cache, table, i32([n]), o, scale=scale)
    want, w = E.tail_want(n, -float(np.float32(scale)))
    kind, count = E.parts_of(dtype, out)
    limit = E.tail_bound(n, w, want, kind, count)
    limit += P.half_step(out) * (want + limit) + torch.finfo(out).smallest_normal * torch.finfo(out).eps
    assert float((o.cpu().double() - want).abs().max()) <= limit, (want, limit)
    assert ncz.paged.sync_status() == 0


# ---------------------------------------------------------------- host threads

def test_host_threads_share_a_stream_and_a_workspace(ncz):
    """Three threads decode on one stream with one workspace, rows that take a join: every call's
    output is that of the same call alone, bit for bit."""
    import threading

    problems = [P.decode_problem(n, 8, 2, 128, 16, [2500 + 100 * i for i in range(n)], BF16, seed=n) for n in (2, 3, 5)]
    stream = torch.cuda.Stream()
    calls, workspace = [], None
    for pr in problems:
        dev = {n: pr[n].cuda() for n in ("q", "k", "v", "table", "lens")}
        cache = ncz.paged.Cache(dev["k"], dev["v"])
        workspace = ncz.paged.decode_workspace(cache, 8) if workspace is None else workspace
        outs = torch.zeros(100, *pr["q"].shape, dtype=BF16, device="cuda")
        calls.append((dev, cache, pr["scale"], outs))
    want = []
    for dev, cache, scale, outs in calls:
        ncz.paged.decode(dev["q"], cache, dev["table"], dev["lens"], outs[0], scale=scale)
        want.append(outs[0].clone())
        outs[0].zero_()
    torch.cuda.synchronize()
    start, failed = threading.Barrier(3), []

    def work(dev, cache, scale, outs):
        try:
            start.wait()
            for o in outs:
                ncz.paged.decode(dev["q"], cache, dev["table"], dev["lens"], o, scale=scale, workspace=workspace,
                                 stream=stream)
        except Exception as e:  # a thread's exception must fail the test
            failed.append(e)

    threads = [threading.Thread(target=work, args=c) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert failed == []
    for (_, _, _, outs), w in zip(calls, want):
        assert bool((outs == w).all())
