"""The paged-cache entry points from several host threads, on fake devices."""
import ctypes
import threading

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
