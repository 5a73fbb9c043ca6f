"""The paged-cache C ABI on the CPU: refusals (before any launch), grids,
kernels and workspace through the fake driver table, and the wrapper's checks."""
import ctypes
import importlib
import os
import shutil
import subprocess

import pytest

from tests import fake_driver as F

F32, F16, BF16, E4M3 = 0, 1, 2, 3
BASE = 0x1000_0000  # fake device addresses, never dereferenced


def status(ncz, st):
    return ncz.flash.STATUS_NAMES[st]


def cache(ncz, *, pages=40, page=16, kv=8, dim=64, dtype=F16, **over):
    row = kv * dim
    c = ncz.paged._Cache(BASE, BASE + 0x800_0000, None, None, pages, page, kv, dim, page * row, row, dim, page * row,
                         row, dim, dtype)
    for name, value in over.items():
        setattr(c, name, value)
    return c


def decode_desc(ncz, *, batch=4, q_heads=8, dim=64, width=64, q_dtype=F16, o_dtype=F16, device=-1, ws=1 << 30, **over):
    d = ncz.paged._Decode(BASE, BASE + 0x100_0000, None, BASE + 0x200_0000, BASE + 0x300_0000, batch, q_heads, width,
                          width, q_heads * dim, dim, q_heads * dim, dim, 0, 0.125, q_dtype, o_dtype,
                          BASE + 0x4000_0000, ws, device, None)
    for name, value in over.items():
        setattr(d, name, value)
    return d


def append_desc(ncz, *, tokens=10, kv=8, dim=64, dtype=F16, device=-1, **over):
    d = ncz.paged._Append(BASE, BASE + 0x100_0000, BASE + 0x200_0000, tokens, kv * dim, dim, kv * dim, dim, dtype,
                          device, None)
    for name, value in over.items():
        setattr(d, name, value)
    return d


def plan_desc(ncz, *, requests=10, width=32, free=100, capacity=50, page=16, device=-1, **over):
    a = [BASE + i * 0x10_0000 for i in range(11)]
    d = ncz.paged._Plan(*a, requests, width, width, free, capacity, page, device, None)
    for name, value in over.items():
        setattr(d, name, value)
    return d


def run(ncz, what, *structs):
    return status(ncz, getattr(ncz.paged.lib(), what)(*(ctypes.byref(s) for s in structs)))


def labels(ncz, launches):
    return [ncz.driver.kernel_label(x.kernel) for x in launches]


BAD_CACHES = [
    ({"k": None}, "InvalidValue"), ({"v": None}, "InvalidValue"), ({"num_pages": 0}, "InvalidValue"),
    ({"page_size": 0}, "InvalidValue"), ({"kv_heads": 0}, "InvalidValue"), ({"head_dim": 48}, "InvalidValue"),
    ({"head_dim": 256}, "InvalidValue"), ({"dtype": F32}, "InvalidValue"), ({"dtype": 4}, "InvalidValue"),
    ({"k_scale": BASE}, "InvalidValue"),                       # scales belong to e4m3
    ({"k_head_stride": 32}, "InvalidValue"), ({"v_token_stride": 64}, "InvalidValue"),  # rows overlap
    ({"k_page_stride": 0}, "InvalidValue"), ({"num_pages": 1 << 31}, "InvalidValue"),
    ({"k_page_stride": 1 << 41}, "Overflow"), ({"k": BASE + 8}, "Misaligned"), ({"v_page_stride": 8196}, "Misaligned"),
]


@pytest.mark.parametrize("over,want", BAD_CACHES)
def test_bad_caches_are_refused_by_every_call(ncz, fake, over, want):
    c = cache(ncz, **over)
    assert run(ncz, "ncz_paged_validate", c) == want
    assert run(ncz, "ncz_paged_append", c, append_desc(ncz)) == want
    assert run(ncz, "ncz_paged_decode", c, decode_desc(ncz)) == want
    assert fake.launches == []


def test_cache_layouts_accepted(ncz):
    assert run(ncz, "ncz_paged_validate", cache(ncz)) == "Success"
    # heads outermost in a page; K and V interleaved in one array of pages; padded rows
    assert run(ncz, "ncz_paged_validate", cache(ncz, k_token_stride=64, k_head_stride=16 * 64)) == "Success"
    assert run(ncz, "ncz_paged_validate", cache(ncz, k_page_stride=2 * 8192, v_page_stride=2 * 8192,
                                                v=BASE + 8192 * 2)) == "Success"
    assert run(ncz, "ncz_paged_validate", cache(ncz, k_head_stride=72, k_token_stride=576, k_page_stride=9216)) == "Success"
    # dimensions of one element may have any stride
    assert run(ncz, "ncz_paged_validate", cache(ncz, kv=1, k_head_stride=3, v_head_stride=0)) == "Success"
    assert run(ncz, "ncz_paged_validate", cache(ncz, dtype=E4M3, k_scale=BASE)) == "Success"
    assert run(ncz, "ncz_paged_validate", cache(ncz, dim=16)) == "Success"
    assert run(ncz, "ncz_paged_validate", cache(ncz, dim=16, dtype=E4M3)) == "InvalidValue"


@pytest.mark.parametrize("over,want", [
    ({"q": None}, "InvalidValue"), ({"o": None}, "InvalidValue"), ({"seq_lens": None}, "InvalidValue"),
    ({"block_table": None}, "InvalidValue"), ({"q_heads": 12}, "InvalidValue"), ({"q_heads": 0}, "InvalidValue"),
    ({"q_dtype": BF16}, "InvalidValue"), ({"q_dtype": F32}, "InvalidValue"), ({"o_dtype": E4M3}, "InvalidValue"),
    ({"table_stride": 63}, "InvalidValue"), ({"o_head_stride": 32}, "InvalidValue"),
    ({"o_batch_stride": 0}, "InvalidValue"), ({"table_width": 1 << 30, "table_stride": 1 << 30}, "Overflow"),
    ({"q": BASE + 1}, "Misaligned"), ({"o": BASE + 1}, "Misaligned"), ({"workspace": BASE + 8}, "Misaligned"),
    ({"workspace": None}, "OutOfMemory"), ({"workspace_bytes": 1000}, "OutOfMemory"),
    ({"lse": BASE + 2}, "Misaligned"), ({"seq_lens": BASE + 2}, "Misaligned"), ({"block_table": BASE + 1}, "Misaligned"),
    ({"q_head_stride": 1 << 41}, "Overflow"), ({"device": 64}, "InvalidDevice"),
])
def test_decode_refusals(ncz, fake, over, want):
    assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, **over)) == want
    assert fake.launches == []


def test_outputs_over_inputs_are_refused(ncz, fake):
    for over in ({"o": BASE}, {"lse": BASE}, {"lse": BASE + 0x100_0000}):
        assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, **over)) == "InvalidValue"
    one = cache(ncz, v=BASE)  # K and V in one: for decode only
    assert run(ncz, "ncz_paged_append", one, append_desc(ncz)) == "InvalidValue"
    assert fake.launches == []
    assert run(ncz, "ncz_paged_decode", one, decode_desc(ncz)) == "Success"


def test_decode_accepts_transposed_and_broadcast_rows(ncz, fake):
    # o as [q_heads][batch][dim]; one q row for every head
    d = decode_desc(ncz, o_head_stride=4 * 64, o_batch_stride=64, q_head_stride=0)
    assert run(ncz, "ncz_paged_decode", cache(ncz), d) == "Success"
    assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, batch=0, q=None)) == "Success"
    assert len(fake.launches) == 1


@pytest.mark.parametrize("over,want", [
    ({"k": None}, "InvalidValue"), ({"v": None}, "InvalidValue"), ({"slots": None}, "InvalidValue"),
    ({"in_dtype": BF16}, "InvalidValue"), ({"in_dtype": F32}, "InvalidValue"), ({"k": BASE + 1}, "Misaligned"),
    ({"slots": BASE + 4}, "Misaligned"), ({"v_token_stride": 1 << 41}, "Overflow"), ({"tokens": 1 << 31}, "InvalidValue"),
])
def test_append_refusals(ncz, fake, over, want):
    assert run(ncz, "ncz_paged_append", cache(ncz), append_desc(ncz, **over)) == want
    assert fake.launches == []


@pytest.mark.parametrize("over,want", [
    ({"held": None}, "InvalidValue"), ({"added": None}, "InvalidValue"), ({"seq_lens": None}, "InvalidValue"),
    ({"block_table": None}, "InvalidValue"), ({"free_pages": None}, "InvalidValue"), ({"slots": None}, "InvalidValue"),
    ({"free_count": None}, "InvalidValue"), ({"left": None}, "InvalidValue"), ({"page_size": 0}, "InvalidValue"),
    ({"table_stride": 31}, "InvalidValue"), ({"slot_capacity": 1 << 31}, "InvalidValue"),
    ({"table_width": 1 << 28, "table_stride": 1 << 28}, "Overflow"),
    ({"seq_lens": BASE + 8}, "InvalidValue"), ({"seq_lens": BASE + 0x10_0000}, "InvalidValue"),  # over held, added
    ({"held": BASE + 2}, "Misaligned"), ({"slots": BASE + 4}, "Misaligned"), ({"status": BASE + 3}, "Misaligned"),
])
def test_plan_refusals(ncz, fake, over, want):
    assert run(ncz, "ncz_paged_plan", plan_desc(ncz, **over)) == want
    assert fake.launches == []


def test_plan_in_place_runs_one_cluster(ncz, fake):
    """Lengths or the free count in place: another cluster might not have read them."""
    assert run(ncz, "ncz_paged_plan", plan_desc(ncz, capacity=100000)) == "Success"
    assert run(ncz, "ncz_paged_plan", plan_desc(ncz, capacity=100000, seq_lens=BASE)) == "Success"
    d = plan_desc(ncz, capacity=100000)
    d.left = d.free_count
    assert run(ncz, "ncz_paged_plan", d) == "Success"
    assert [x.grid for x in fake.launches] == [128, 8, 8]


def test_at_most_2_to_the_24_requests(ncz, fake):
    """The kernels count requests, rounded up to whole rounds, in 32 bits."""
    wide = {"seq_lens": BASE + (1 << 36), "added": BASE + (1 << 40)}
    assert run(ncz, "ncz_paged_plan", plan_desc(ncz, requests=1 << 24, **wide)) == "Success"
    assert len(fake.launches) == 1
    for n in ((1 << 24) + 1, (1 << 31) - 1):
        assert run(ncz, "ncz_paged_plan", plan_desc(ncz, requests=n, **wide)) == "InvalidValue"
        assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, batch=n)) == "InvalidValue"
    assert len(fake.launches) == 1


def test_plan_without_optional_outputs(ncz, fake):
    assert run(ncz, "ncz_paged_plan", plan_desc(ncz, positions=None, starts=None, status=None)) == "Success"
    assert run(ncz, "ncz_paged_plan", plan_desc(ncz, requests=0, held=None, added=None, seq_lens=None,
                                                block_table=None)) == "Success"
    assert labels(ncz, fake.launches) == ["paged_plan"] * 2
    assert all(x.grid % 8 == 0 for x in fake.launches)  # whole clusters


def test_decode_kernels_by_type_and_group(ncz, fake):
    for dtype, name in ((F16, "f16"), (BF16, "bf16"), (E4M3, "e4m3")):
        for dim in (16, 32, 64, 128):
            if dtype == E4M3 and dim == 16:
                continue
            for group, rows in ((1, 1), (8, 1), (9, 2), (16, 2), (17, 4), (40, 4)):
                fake.launches.clear()
                d = decode_desc(ncz, q_heads=2 * group, dim=dim, q_dtype=BF16 if dtype == BF16 else F16, batch=100,
                                o_dtype=F32)
                assert run(ncz, "ncz_paged_decode", cache(ncz, kv=2, dim=dim, dtype=dtype), d) == "Success"
                assert labels(ncz, fake.launches) == [f"paged_decode<{dim},{name},{rows}>", f"paged_join<{dim}>"]


def test_decode_kernel_for_few_short_rows(ncz, fake):
    """A cluster of eight CTAs a row where rows are few and short, no join; else the even shares."""
    def first(kv, group, batch, keys, dim=128, dtype=BF16, **kw):
        fake.launches.clear()
        d = decode_desc(ncz, q_heads=kv * group, dim=dim, q_dtype=F16 if dtype == F16 else BF16, batch=batch,
                        width=keys // 16, **kw)
        assert run(ncz, "ncz_paged_decode", cache(ncz, kv=kv, dim=dim, dtype=dtype), d) == "Success"
        return labels(ncz, fake.launches)

    assert first(8, 4, 1, 1024) == ["paged_decode_few<128,bf16,1>"] and fake.launches[0].grid == 64
    assert first(8, 12, 1, 1024) == ["paged_decode_few<128,bf16,2>"]
    assert first(8, 4, 4, 1024) == ["paged_decode_few<128,bf16,1>"] and fake.launches[0].grid == 256
    assert first(8, 8, 1, 1024, dtype=E4M3) == ["paged_decode_few<128,e4m3,1>"]
    assert first(1, 1, 1, 1024, 16, F16) == ["paged_decode_few<16,f16,1>"]
    assert first(8, 4, 1, 16384, window=1000) == ["paged_decode_few<128,bf16,1>"]
    assert first(8, 4, 1, 4096) == ["paged_decode<128,bf16,1>", "paged_join<128>"]  # too long
    assert first(8, 4, 5, 1024)[0] == "paged_decode<128,bf16,1>"                     # too many
    assert first(8, 20, 1, 1024)[0] == "paged_decode<128,bf16,4>"                    # two warps a slice of keys
    assert first(8, 4, 1, 64) == ["paged_decode<128,bf16,1>"]                        # one tile


def test_decode_kernel_for_many_heads_per_kv_head(ncz, fake):
    """The tcgen05 kernel: 16-bit caches, head_dim 64 or 128, enough query heads and
    steps of 128 keys, 16-bit outputs; one CTA per SM."""
    def label(dim, group, dtype=BF16, o_dtype=BF16, batch=64, width=64, kv=1):
        fake.launches.clear()
        q_dtype = BF16 if dtype == E4M3 else dtype
        d = decode_desc(ncz, q_heads=kv * group, dim=dim, q_dtype=q_dtype, o_dtype=o_dtype, batch=batch, width=width)
        assert run(ncz, "ncz_paged_decode", cache(ncz, kv=kv, dim=dim, dtype=dtype), d) == "Success"
        return labels(ncz, fake.launches)[0]

    assert label(64, 17) == "paged_decode_wide<64,bf16,32>" and fake.launches[0].grid == 148
    assert label(64, 33, F16, F16) == "paged_decode_wide<64,f16,64>"
    assert label(128, 65) == "paged_decode_wide<128,bf16,128>" and label(128, 300) == "paged_decode_wide<128,bf16,128>"
    assert label(128, 9) == "paged_decode_wide<128,bf16,32>" and label(64, 16) == "paged_decode<64,bf16,2>"
    assert label(128, 8) == "paged_decode<128,bf16,1>"
    for other in (label(32, 32), label(128, 32, E4M3), label(128, 32, o_dtype=F32), label(128, 32, batch=30),
                  label(128, 32, width=24)):
        assert other.startswith("paged_decode<")
    assert label(128, 32, batch=4, kv=8, width=96).startswith("paged_decode_wide<")
    # tensor memory's sums are kept short beside the output's rounding: steps of one row in one CTA
    assert label(64, 32, F16, F16, batch=1000, width=1024 * 8).startswith("paged_decode_wide<")
    assert label(64, 32, F16, F16, batch=1000, width=1025 * 8).startswith("paged_decode<")
    assert label(64, 32, F16, F16, batch=10, width=1025 * 8).startswith("paged_decode_wide<")
    assert label(64, 32, batch=1000, width=1025 * 8).startswith("paged_decode_wide<")
    assert label(64, 32, batch=1000, width=8193 * 8).startswith("paged_decode<")


def test_status_word_and_hooks(ncz, fake):
    lib = ncz.paged.lib()
    assert ncz.paged.sync_status(3) == 0
    fake.symbol_words[3] = 0x81000005
    assert status(ncz, lib.ncz_paged_sync_status(3)) == "DeviceTimeout"
    assert ncz.paged.sync_status(3) == 0 and fake.current() == 0
    assert lib.ncz_paged_test_set_wait_limit(2, 5) == 0 and lib.ncz_paged_test_drop_scores(2, 1) == 0
    assert [(dev, len(x)) for dev, x in fake.symbol_writes[-2:]] == [(2, 8), (2, 4)]


def test_decode_grid_and_join(ncz, fake):
    # 64 * 16 keys at most: the grid is what is resident at once, in whole sets of the 8 heads
    assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, batch=100)) == "Success"
    grid = fake.launches[0].grid
    assert grid % 8 == 0 and 148 <= grid <= 148 * 16 and fake.launches[1].grid == grid
    fake.launches.clear()
    # a table of one page: one CTA per row, each whole in it, nothing to join
    assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, batch=3, width=1)) == "Success"
    assert labels(ncz, fake.launches) == ["paged_decode<64,f16,1>"] and fake.launches[0].grid == 24
    # a head count that would leave CTAs without work: the tiles in one list
    fake.launches.clear()
    assert run(ncz, "ncz_paged_decode", cache(ncz, kv=300), decode_desc(ncz, batch=100, q_heads=300)) == "Success"
    assert fake.launches[0].grid >= grid
    fake.launches.clear()
    # few long rows: join blocks for each of the 8 rows
    assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, batch=1, q_heads=32, width=512)) == "Success"
    assert fake.launches[1].grid % 8 == 0
    # a window bounds the keys too
    fake.launches.clear()
    assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, batch=1, window=100)) == "Success"
    assert labels(ncz, fake.launches) == ["paged_decode<64,f16,1>"]


def test_workspace_holds_every_launch(ncz, fake):
    need = ctypes.c_size_t(0)
    c = cache(ncz)
    lib = ncz.paged.lib()
    assert lib.ncz_paged_decode_workspace(ctypes.byref(c), 8, 3, ctypes.byref(need)) == 0
    # 2 parts per CTA of 8 rows of 64 + 2 floats, and a record per CTA
    assert run(ncz, "ncz_paged_decode", c, decode_desc(ncz, batch=100)) == "Success"
    grid = fake.launches[0].grid
    assert need.value >= grid * 16 + 2 * grid * 8 * 66 * 4
    assert run(ncz, "ncz_paged_decode", c, decode_desc(ncz, ws=need.value)) == "Success"
    assert run(ncz, "ncz_paged_decode", c, decode_desc(ncz, ws=need.value - 1)) == "OutOfMemory"
    assert status(ncz, lib.ncz_paged_decode_workspace(ctypes.byref(c), 12, -1, ctypes.byref(need))) == "InvalidValue"
    assert status(ncz, lib.ncz_paged_decode_workspace(ctypes.byref(c), 8, -1, None)) == "InvalidValue"


def test_launches_go_to_the_named_device_and_count(ncz, fake):
    before = ncz.flash.launch_count()
    assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, device=5)) == "Success"
    assert run(ncz, "ncz_paged_append", cache(ncz), append_desc(ncz, device=2)) == "Success"
    assert run(ncz, "ncz_paged_plan", plan_desc(ncz, device=7)) == "Success"
    assert [x.device for x in fake.launches] == [5, 2, 7] and fake.current() == 0
    assert ncz.flash.launch_count() - before == 3


def test_failures_reach_the_caller(ncz, fake):
    fake.fail("set_max_dynamic_smem", device=3, error=F.INVALID_VALUE)
    assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, device=3)) == "InvalidValue"
    assert fake.launches == [] and fake.current() == 0
    assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, device=3)) == "Success"
    fake.launches.clear()
    fake.fail("launch_kernel", device=3, error=F.LAUNCH_FAILURE)
    assert run(ncz, "ncz_paged_decode", cache(ncz), decode_desc(ncz, device=3)) == "LaunchFailed"
    assert fake.launches == []  # no join without its decode
    fake.fail("set_device", device=4, error=F.INVALID_DEVICE)
    assert run(ncz, "ncz_paged_append", cache(ncz), append_desc(ncz, device=4)) == "InvalidDevice"
    assert fake.current() == 0


def test_wrapper_refuses_host_tensors(ncz):
    torch = pytest.importorskip("torch")
    pages = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(ncz.FlashError, match="CUDA"):
        ncz.paged.Cache(pages, pages.clone())
    ints = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ncz.FlashError, match="CUDA"):
        ncz.paged.plan(ints, ints, ints, ints[:1], ints.view(2, 2), ints, torch.zeros(4, dtype=torch.int64), page_size=16)


@pytest.mark.parametrize("compiler,lang", [("gcc", ["-std=c99"]), ("g++", ["-std=c++17", "-x", "c++"])])
def test_header_from_c_and_cpp(ncz, tmp_path, compiler, lang):
    """include/ncz_paged.h as C99 and C++17 without warnings, refusals before any
    device call (tests/c_abi/paged_consumer.c)."""
    cc = shutil.which(compiler)
    if cc is None:
        pytest.skip(f"no {compiler}")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    libdir = os.path.dirname(ncz.flash.LIB_PATH)
    exe = tmp_path / "paged_consumer"
    build = subprocess.run([cc] + lang + ["-Wall", "-Wextra", "-Werror", "-pedantic", "-I", os.path.join(root, "include"),
                                          os.path.join(root, "tests", "c_abi", "paged_consumer.c"), "-x", "none", "-L",
                                          libdir, "-lncz_flash", f"-Wl,-rpath,{libdir}", "-o", str(exe)],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    ran = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert ran.returncode == 0 and "paged consumer: ok" in ran.stdout, ran.stderr


def test_struct_sizes_match_the_header(ncz, tmp_path):
    """The ctypes mirrors have the sizes and last offsets that the C compiler gives the header's structs."""
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no gcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = [("ncz_paged_cache", "dtype"), ("ncz_paged_plan_desc", "stream"), ("ncz_paged_append_desc", "stream"),
              ("ncz_paged_decode_desc", "stream"), ("ncz_paged_decode_desc", "workspace")]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "ncz_paged.h"\nint main(void) {\n' + "".join(
        f'    printf("%zu %zu\\n", sizeof({s}), offsetof({s}, {f}));\n' for s, f in fields) + "    return 0;\n}\n")
    exe = tmp_path / "sizes"
    subprocess.run([cc, "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [tuple(int(x) for x in line.split()) for line in
           subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()]
    pg = ncz.paged
    mirrors = [pg._Cache, pg._Plan, pg._Append, pg._Decode, pg._Decode]
    assert got == [(ctypes.sizeof(m), getattr(m, f).offset) for m, (_, f) in zip(mirrors, fields)]


def test_compare_takes_paged_shapes(ncz, monkeypatch):
    compare = importlib.import_module("not-cute-zig_b200.compare")
    seen = []
    monkeypatch.setattr(compare, "compare_paged", lambda n, *a: seen.append(a) or {"correct": True})
    assert compare.main(["--paged-shape", "2,8,4,64,100,f16"]) == 0 and seen == [(2, 8, 4, 64, 100, "f16")]
    assert compare.main(["--paged"]) == 0 and seen[1:] == compare.PAGED_SHAPES
