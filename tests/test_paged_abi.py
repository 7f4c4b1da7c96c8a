"""libinfiniop_paged.so without a GPU: its symbols and header, and every check
that a create function makes, reached with a hand-made handle (a plain struct of
which the create functions read fields only)."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import operators_amd as oa
from operators_amd.liboperators import PAGED_LIB_NAME, PAGED_SYMBOLS, library_path

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, PARAM, DTYPE, SHAPE, STRIDES, MEMORY, DEVICE = 0, 2, 3, 4, 5, 6, 8


class FakeHandle(ctypes.Structure):
    _fields_ = [("device", ctypes.c_int), ("device_id", ctypes.c_int), ("cu_count", ctypes.c_int), ("lds", ctypes.c_int),
                ("grid", ctypes.c_int), ("wave", ctypes.c_int)]


def declared():
    text = open(os.path.join(ROOT, "include", "infiniop_paged.h")).read()
    return sorted(set(re.findall(r"INFINIOP_EXPORT\s+infiniopStatus_t\s+(infiniop\w+)\s*\(", text)))


def test_library_exports_what_the_header_declares():
    assert sorted(PAGED_SYMBOLS) == declared()
    out = subprocess.run(["nm", "-D", "--defined-only", library_path(PAGED_LIB_NAME)], capture_output=True, text=True, check=True).stdout
    exported = sorted(line.split()[-1] for line in out.splitlines() if re.search(r"\s[TtDdBbWwVv]\s", line))
    assert [s for s in exported if s.startswith("infiniop")] == declared()
    assert [s for s in exported if not s.startswith(("infiniop", "_init", "_fini", "__hip", "_edata", "_end", "__bss_start"))] == []


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_header_is_plain_c(tmp_path):
    tu = tmp_path / "one.c"
    tu.write_text('#include "infiniop_paged.h"\nint main(void) { infiniopPagedAttentionDescriptor_t d = 0; return d != 0 || F8E4M3.mantissa != 3; }\n')
    for cmd in (["gcc", "-std=c11"], ["g++", "-std=c++17", "-x", "c++"]):
        res = subprocess.run(cmd + ["-Wall", "-Wextra", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(tu)], capture_output=True, text=True)
        assert res.returncode == 0, res.stderr


def test_float8_has_a_layout():
    from operators_amd.utils import torch_dtype_to_layout

    assert torch_dtype_to_layout(torch.float8_e4m3fn) == oa.F8E4M3
    assert int.from_bytes(bytes(oa.F8E4M3), "little") == 1 | (1 << 8) | (1 << 9) | (3 << 16) | (4 << 24)




def spec(t):
    return t if isinstance(t, tuple) else (tuple(t.shape), tuple(t.stride()), t.dtype)


def create(op, tensors, *params, device=4, desc=True):
    """The status of a create call on (shape, strides, dtype) triples; destroys what it made."""
    from operators_amd import liboperators as lo
    from operators_amd.utils import make_descriptor, torch_dtype_to_layout

    lib, base = oa.open_paged_lib(), oa.open_lib()
    handle = FakeHandle(device, 0, 256, 163840, 2 ** 31 - 1, 64)
    made = [make_descriptor(base, s, st, torch_dtype_to_layout(dt)) for s, st, dt in map(spec, tensors)]
    d = getattr(lo, f"infiniop{op}Descriptor_t")()
    h = ctypes.cast(ctypes.pointer(handle), lo.infiniopHandle_t)
    status = getattr(lib, f"infiniopCreate{op}Descriptor")(h, ctypes.byref(d) if desc else None, *made, *params)
    for m in made:
        base.infiniopDestroyTensorDescriptor(m)
    size = None
    if status == OK:
        ask = getattr(lib, f"infiniopGet{op}WorkspaceSize", None)
        if ask is not None:
            n = ctypes.c_uint64(0)
            assert ask(d, ctypes.byref(n)) == OK and ask(d, None) == PARAM
            size = n.value
        assert getattr(lib, f"infiniopDestroy{op}Descriptor")(d) == OK
    return status if size is None else (status, size)


def dense(shape, dtype):
    st, run = [], 1
    for n in reversed(shape):
        st.append(run)
        run *= n
    return tuple(shape), tuple(reversed(st)), dtype


I32, F16, F32, I8, E4M3 = torch.int32, torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn


def cache(pages=10, heads=2, page=32, dim=64, blocks=2, dtype=I8):
    c, s = dense((pages, heads, page, dim), dtype), dense((pages, heads, blocks), F32)
    return [c, c, s, s]


def batch(rows=3, cols=4):
    return [dense((rows, cols), I32), dense((rows + 1,), I32), dense((rows,), I32)]


def append_args(**more):
    x = dense((5, more.get("heads", 2), more.get("dim", 64)), F16)
    return cache(**more) + [x, x] + batch()


def attention_args(heads=4, **more):
    x = dense((5, heads, more.get("dim", 64)), F16)
    return [x, x] + cache(**more) + batch()


OPS = {
    "KVCacheAppend": (append_args, ()),
    "PagedAttention": (attention_args, (1, 0.125)),
    "KVCacheCopy": (lambda **m: cache(**m) + [dense((7, 2), I32)], ()),
}


def status(op, tensors, *params, **more):
    got = create(op, tensors, *(params or OPS[op][1]), **more)
    return got[0] if isinstance(got, tuple) else got


@pytest.mark.parametrize("op", OPS)
def test_common_refusals(op):
    args, params = OPS[op]
    assert status(op, args()) == OK
    assert status(op, args(dtype=E4M3)) == OK
    for other in (0, 1, 2, 3, 17):
        assert status(op, args(), device=other) == DEVICE
    assert status(op, args(), desc=False) == MEMORY
    lib = oa.open_paged_lib()
    assert getattr(lib, f"infiniopDestroy{op}Descriptor")(None) == PARAM


@pytest.mark.parametrize("op", OPS)
def test_null_arguments(op):
    from operators_amd import liboperators as lo

    args, params = OPS[op]
    lib = oa.open_paged_lib()
    n = len(args())
    d = getattr(lo, f"infiniop{op}Descriptor_t")()
    assert getattr(lib, f"infiniopCreate{op}Descriptor")(None, ctypes.byref(d), *([None] * n), *params) == PARAM
    handle = FakeHandle(4, 0, 256, 163840, 2 ** 31 - 1, 64)
    h = ctypes.cast(ctypes.pointer(handle), lo.infiniopHandle_t)
    assert getattr(lib, f"infiniopCreate{op}Descriptor")(h, ctypes.byref(d), *([None] * n), *params) == PARAM
    pointers = {"KVCacheAppend": 12, "PagedAttention": 12, "KVCacheCopy": 6}[op]
    assert getattr(lib, f"infiniop{op}")(None, *([None] * (1 if pointers == 12 else 0)), *([0] if pointers == 12 else []), *([None] * (10 if pointers == 12 else 6))) == PARAM


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("change, want", [
    (dict(dim=24), SHAPE), (dict(dim=272), SHAPE), (dict(dim=256), OK), (dict(dim=16), OK),
    (dict(page=24, blocks=1), SHAPE), (dict(page=48, blocks=3), OK), (dict(page=48, blocks=2), SHAPE), (dict(page=32, blocks=4), SHAPE),
    (dict(page=32, blocks=1), OK), (dict(pages=0), SHAPE), (dict(pages=1), OK), (dict(heads=1), OK),
    (dict(dtype=torch.uint8), DTYPE), (dict(dtype=torch.float16), DTYPE),
])
def test_cache_shapes(op, change, want):
    if op == "PagedAttention" and change.get("heads") == 1:
        assert status(op, attention_args(heads=3, **{k: v for k, v in change.items() if k != "heads"})[:2] + cache(heads=1) + batch()) == OK
        return
    assert status(op, OPS[op][0](**change)) == want


@pytest.mark.parametrize("op", OPS)
def test_cache_strides_and_mixed_types(op):
    at = {"KVCacheAppend": 0, "PagedAttention": 2, "KVCacheCopy": 0}[op]

    def with_(i, t):
        a = OPS[op][0]()
        a[at + i] = t
        return status(op, a)

    shape = (10, 2, 32, 64)
    assert with_(1, (shape, (8192, 4096, 128, 1), I8)) == OK          # rows of codes in a wider buffer
    assert with_(1, (shape, (8192, 64, 128, 1), I8)) == OK            # heads inside tokens
    assert with_(0, (shape, (4096, 2048, 64, 2), I8)) == STRIDES
    assert with_(0, (shape, (4096, 2048, 72, 1), I8)) == STRIDES      # not a multiple of 16
    assert with_(0, (shape, (4096, 2056, 64, 1), I8)) == STRIDES
    assert with_(0, (shape, (4104, 2048, 64, 1), I8)) == STRIDES
    assert with_(0, (shape, (4096, 2048, 48, 1), I8)) == STRIDES      # tokens that overlap
    assert with_(0, (shape, (4096, 0, 64, 1), I8)) == STRIDES
    assert with_(0, (shape, (-4096, 2048, 64, 1), I8)) == STRIDES
    assert with_(0, (shape, (1 << 40, 1 << 31, 64, 1), I8)) == STRIDES  # a page that spans 2^31
    assert with_(0, (shape, (1 << 40, 2048, 64, 1), I8)) == OK
    assert with_(1, dense(shape, E4M3)) == DTYPE
    assert with_(1, dense((10, 2, 64, 64), I8)) == SHAPE
    assert with_(2, dense((10, 2, 2), torch.float16)) == DTYPE
    assert with_(3, dense((10, 2, 1), F32)) == SHAPE
    assert with_(3, dense((9, 2, 2), F32)) == SHAPE
    assert with_(3, dense((10, 4), F32)) == SHAPE
    assert with_(2, ((10, 2, 2), (8, 4, 2), F32)) == STRIDES
    assert with_(2, ((10, 2, 2), (8, 4, 1), F32)) == OK


@pytest.mark.parametrize("op", ["KVCacheAppend", "PagedAttention"])
def test_batch_and_tokens(op):
    n = len(OPS[op][0]())

    def with_(i, t):
        a = OPS[op][0]()
        a[i] = t
        return status(op, a)

    assert with_(n - 3, dense((3, 4), torch.int64)) == DTYPE
    assert with_(n - 3, ((3, 4), (9, 1), I32)) == OK
    assert with_(n - 3, ((3, 4), (3, 1), I32)) == STRIDES
    assert with_(n - 3, ((3, 4), (8, 2), I32)) == STRIDES
    assert with_(n - 3, dense((3, 0), I32)) == SHAPE
    assert with_(n - 3, dense((3, 1 << 27), I32)) == SHAPE      # 2^32 places
    assert with_(n - 3, dense((12,), I32)) == SHAPE
    assert with_(n - 2, dense((3,), I32)) == SHAPE
    assert with_(n - 2, ((4,), (2,), I32)) == STRIDES
    assert with_(n - 1, dense((4,), I32)) == SHAPE
    x = 0 if op == "PagedAttention" else 4
    heads = 4 if op == "PagedAttention" else 2
    assert with_(x, dense((5, heads, 64), F32)) == DTYPE
    assert with_(x, dense((5, heads, 64), torch.bfloat16)) == DTYPE  # the other one is fp16
    assert with_(x, dense((6, heads, 64), F16)) == SHAPE
    assert with_(x, dense((5, heads, 48), F16)) == SHAPE
    assert with_(x, ((5, heads, 64), (1024, 128, 2), F16)) == STRIDES
    assert with_(x, ((5, heads, 64), (1031, 67, 1), F16)) == OK
    # no tokens, no rows: nothing to do
    a = OPS[op][0]()
    empty = [dense((0, heads, 64), F16)] * 2
    a[x:x + 2] = empty
    assert status(op, a) == OK
    a[n - 3:] = batch(rows=0)
    assert status(op, a) == OK


def test_attention_parameters():
    assert status("PagedAttention", attention_args(heads=5)) == SHAPE      # not a multiple of the two K/V heads
    assert status("PagedAttention", attention_args(), 0, 0.1) == PARAM
    assert status("PagedAttention", attention_args(), 1, float("nan")) == PARAM
    assert status("PagedAttention", attention_args(), 1, float("inf")) == PARAM
    got, size = create("PagedAttention", attention_args(), 1, 0.1)
    assert got == OK and 0 < size < 1 << 28


@pytest.mark.parametrize("rows, cols, tokens, most, heads, kv, dim", [
    (2, 2, 200, 100, 64, 8, 128), (2, 64, 200, 100, 64, 8, 128), (1, 4, 1, 1, 32, 8, 128), (1, 3, 90, 90, 8, 1, 64), (300, 8, 300, 1, 8, 1, 64), (5, 5, 40, 8, 8, 512, 256),
    (3, 4096, 100, 100, 8, 1, 128)])
def test_attention_workspace(rows, cols, tokens, most, heads, kv, dim):
    """Room for no more parts than the rows' tiles can be cut into with tables of that length, nor than the GPU's units make of them."""
    heads = max(heads, kv)
    x = dense((tokens, heads, dim), F16)
    got, size = create("PagedAttention", [x, x] + cache(pages=4, heads=kv, page=16, dim=dim, blocks=1) + batch(rows=rows, cols=cols), most, 0.1)
    assert got == OK
    steps, query, room = -(-cols * 16 // 32), most * heads // kv, 16
    for tile, least, upto, units in ((16 if query <= 16 or dim > 128 else 32, 4 if rows == 1 else 8, 64, 4 * 256), (256 if dim <= 128 else 128, 16, query, 3 * 256)):
        chunks = -(-steps // least)
        slots = min(rows * -(-min(query, upto) // tile) * (chunks if chunks > 1 else 0), 2 * -(-units // kv) + 6)
        room = max(room, slots * kv * tile * (dim + 2) * 4)
    assert 0 < size <= room


def test_copy_pairs():
    assert status("KVCacheCopy", cache() + [dense((7, 3), I32)]) == SHAPE
    assert status("KVCacheCopy", cache() + [dense((7, 2), torch.int64)]) == DTYPE
    assert status("KVCacheCopy", cache() + [((7, 2), (4, 1), I32)]) == STRIDES
    assert status("KVCacheCopy", cache() + [dense((0, 2), I32)]) == OK


def update_args(rows=3, cols=4, pages=20):
    t, r, p = dense((rows, cols), I32), dense((rows,), I32), dense((pages,), I32)
    return [t, r, p, dense((rows, 2), I32), dense((2,), I32), t, r, p, r, r]


def compact_args(rows=3, cols=4, pages=20):
    t, r, p = dense((rows, cols), I32), dense((rows,), I32), dense((pages,), I32)
    return [t, p, dense((pages // 2, 2), I32), dense((2,), I32), t, r, p]


@pytest.mark.parametrize("op, args", [("PageTableUpdate", update_args), ("PageTableCompact", compact_args)])
def test_page_table_refusals(op, args):
    def status_of(a, page=16, **more):
        got = create(op, a, page, **more)
        return got[0] if isinstance(got, tuple) else got

    assert status_of(args()) == OK
    assert status_of(args(rows=8192)) == OK
    assert status_of(args(rows=8193)) == SHAPE
    assert status_of(args(pages=(1 << 24) - 1)) == OK
    assert status_of(args(pages=1 << 24)) == SHAPE
    assert status_of(args(), page=0) == PARAM
    assert status_of(args(), page=1 << 20) == PARAM
    assert status_of(args(), page=1) == OK
    assert status_of(args(), device=0) == DEVICE
    assert status_of(args(), desc=False) == MEMORY
    for i in range(len(args())):
        a = args()
        s, st, _ = a[i]
        a[i] = (s, st, torch.int64)
        assert status_of(a) == DTYPE, i
        a[i] = dense(s[:-1] + (s[-1] + 1,), I32)
        assert status_of(a) == SHAPE, i
        a[i] = (s, st[:-1] + (2,), I32)
        assert status_of(a) == STRIDES, i
    a = args()
    a[2 if op == "PageTableCompact" else 3] = dense((2, 2), I32)  # too short a list
    assert status_of(a) == SHAPE
    lib = oa.open_paged_lib()
    assert getattr(lib, f"infiniopDestroy{op}Descriptor")(None) == PARAM
    assert getattr(lib, f"infiniopGet{op}WorkspaceSize")(None, None) == PARAM


def run_cc(tmp_path, body):
    """The lines that a host program on the library's own header prints."""
    tu, exe = tmp_path / "one.cc", tmp_path / "one"
    tu.write_text('#include "paged/paged_attention/amd/paged_attention_amd.h"\n#include <cstdio>\n#include <cstdlib>\n' + body)
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    res = subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "operators_amd", "csrc"),
                          "-isystem", os.path.join(rocm, "include"), str(tu), "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    return lambda *args: subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True, check=True).stdout.split()


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_units_of_rows_that_are_long_together(tmp_path):
    """How long a unit of attention is, as the kernels work it out, where the rows' steps exceed 2^32 together: 64 rows of 2^31 places
    and one unit to be made of each of 256 K/V heads.  A number that wrapped around would cut them into more units than the grid
    and the workspace have room for."""
    unit_steps = run_cc(tmp_path, '''int main(int n, char **v) {
    for (int i = 1; i + 2 < n; i += 3) std::printf("%u\\n", paged_unit_steps(std::strtof(v[i], nullptr), std::atoi(v[i + 1]), std::atoi(v[i + 2])));
}
''')
    wanted = [0.0, 0.5, 7.0, 15.9, 16.0, 100.5, 2.0 ** 20, 2.0 ** 26, 2.0 ** 29 + 64, 2.0 ** 30, 2.0 ** 31, 2.0 ** 32 - 256, 2.0 ** 32, 1.5 * 2.0 ** 32, 2.0 ** 40, 1e30]
    for least, whole in ((4, 1), (8, 1), (16, 2)):
        out = unit_steps(*[x for w in wanted for x in (w, least, whole)])
        for w, steps in zip(wanted, map(int, out)):
            assert steps >= least and steps % whole == 0 and steps >= min(w, 2 ** 30) and steps <= max(w + 2, least, 2) and steps <= 2 ** 30, (w, steps)
    total, longest = 64 * 2 ** 26, 2 ** 26
    for by in (1.5, 1.25, 1.0, 2 / 3, 0.5, 1 / 3):
        out = int(unit_steps(total * by * 1.00001, 16, 2)[0])
        units = 64 * -(-longest // out)
        assert units <= 64 + total / (total * by) and (units == 64 or units <= 2 * total / (total * by)), by


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_sums_over_rows_that_name_the_same_tokens(tmp_path):
    """Offsets that rise and fall again give half of all rows all tokens.  131072 such rows of 32768 tiles are 2^32 units, 2^24 rows of
    nearly 2^24 tiles of 2^26 steps more work than 64 bits hold: no sum of units reaches that of the slots, and no sum of work wraps."""
    sums = run_cc(tmp_path, '''int main() {
    uint64_t all = 0;
    for (int lane = 0; lane < 512; ++lane) {
        uint64_t mine = 0;
        for (int r = 0; r < 256; ++r) mine += PagedSum::both(32768, 0);
        all += mine;
    }
    all += PagedSum::both(7, 1535);
    std::printf("%llu %u\\n", (unsigned long long)PagedSum::units(all), PagedSum::slots(all));
    uint64_t total = 0;
    for (int lane = 0; lane < 512; ++lane) {
        uint64_t mine = 0;
        for (int r = 0; r < 32768; ++r) mine = PagedSum::work(mine, (1u << 24) - 1, 1u << 26);
        total += mine;
    }
    std::printf("%llu\\n", (unsigned long long)total);
    std::printf("%llu %llu\\n", (unsigned long long)PagedSum::work(5, 3, 1000), (unsigned long long)PagedSum::work((1ull << 54) - 1, 1, 1));
}
''')
    assert [int(x) for x in sums()] == [2 ** 32 + 7, 1535, 2 ** 63, 3005, 2 ** 54]


def test_no_fallback():
    with pytest.raises(FileNotFoundError):
        oa.open_paged_lib("/nonexistent/libinfiniop_paged.so")
