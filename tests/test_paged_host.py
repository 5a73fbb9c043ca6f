"""The paged-cache entry points from several host threads, on fake devices, and what the
GPU tests' rounding bounds can tell apart."""
import ctypes
import threading

import torch

from tests import paged_edge_cases as E
from tests.test_paged import BASE, cache, decode_desc, labels


def test_decodes_of_two_threads_on_one_stream_keep_their_joins(ncz, fake):
    """Calls on one stream may share a workspace: a second thread's decode never comes between
    the first one's decode kernel and the join that reads what it left."""
    table, c, status = fake.table(), cache(ncz), []
    stream = BASE + 64
    calls = [decode_desc(ncz, batch=n, width=256, stream=stream) for n in (30, 40)]

    def decode(d):
        status.append(ncz.paged.lib().ncz_paged_decode(ctypes.byref(c), ctypes.byref(d)))

    second = threading.Thread(target=decode, args=(calls[1],))
    plain, first = table["launch_kernel"], []

    def launch(*args):
        e = plain(*args)
        if not first:
            first.append(True)
            second.start()
            second.join(0.5)  # time enough to pass, were it let
        return e

    table["launch_kernel"] = launch
    assert ncz.driver.install(table) == 0
    decode(calls[0])
    second.join()
    assert status == [0, 0]
    names = labels(ncz, fake.launches)
    assert [n.split("<")[0] for n in names] == ["paged_decode", "paged_join"] * 2
    assert {x.stream for x in fake.launches} == {stream}


def test_the_two_key_rows_tell_the_parts_of_p_apart():
    """The bound that tests/test_paged_edges_gpu.py holds f32 outputs to is below the error that
    one part fewer would give, and above that of the parts there are."""
    for dtype in (E.F16, E.BF16, E.E4M3):
        kind, count = E.parts_of(dtype, E.F32)
        p = 256 * torch.exp(E.two_keys(dtype).double())
        error = lambda n: float(((E.in_parts(p, kind, n) - p).abs() / p).max())  # noqa: E731
        assert error(count) <= E.weight_error(kind, count)[0] + 2.0 ** -24
        assert error(count - 1) > 1.5 * E.TWO_KEYS_BOUND


def test_scale_zero_takes_the_warp_mmas(ncz, fake):
    """They alone turn Q into 0 times itself."""
    c = cache(ncz, kv=1)
    for scale, kernel in ((0.125, "paged_decode_wide"), (-0.125, "paged_decode_wide"), (1e-45, "paged_decode_wide"),
                          (0.0, "paged_decode"), (-0.0, "paged_decode")):
        fake.launches.clear()
        d = decode_desc(ncz, q_heads=32, batch=64, scale=scale)
        assert ncz.paged.lib().ncz_paged_decode(ctypes.byref(c), ctypes.byref(d)) == 0
        assert labels(ncz, fake.launches)[0].split("<")[0] == kernel, scale
