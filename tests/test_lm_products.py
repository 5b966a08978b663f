"""Products of quantised language models: 4-bit matrix-vector products, int8 products grouped by
expert, and the plan that groups slots by expert.  Everything is integer arithmetic with one right
answer, so every comparison is for equality with numpy's int64 (tolerance zero: each output is the
exact sum, or its low 64 bits, shifted and truncated once)."""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

import mind_b200
from mind_b200 import blas

I32 = np.int32
CANARY = 0x5A5A5A5A


# ------------------------------------------------------------------- plain implementations
def low32(v):
    return (v.astype(np.int64) & 0xFFFFFFFF).astype(np.uint32).view(np.int32)


def unpack4(w, cols):
    """(…, pitch) int8 -> (…, cols) int64, even column in the low half."""
    b = w.astype(np.int64) & 255
    d = np.stack([b & 15, b >> 4], axis=-1).reshape(*w.shape[:-1], -1)
    return ((d ^ 8) - 8)[..., :cols]


def ref_w4(w, scale, x, cols, group, shift):
    """int64 throughout; numpy's int64 wraps mod 2^64, as the definition does."""
    d = unpack4(w, cols)
    total = np.zeros((x.shape[0], w.shape[0]), np.int64)
    with np.errstate(over="ignore"):
        for g in range(scale.shape[1]):
            k0, k1 = g * group, min(cols, (g + 1) * group)
            total += (x[:, k0:k1].astype(np.int64) @ d[:, k0:k1].T) * scale[:, g].astype(np.int64)
    return low32(total >> shift)


def gather(x, rows_of, p, width):
    out = np.zeros((len(p), width), np.int64)
    for j, q in enumerate(p):
        r = q if rows_of is None else rows_of[q]
        if 0 <= r < x.shape[0]:
            out[j] = x[r]
    return out


def ref_w4_grouped(w, scale, x, rows_of, offsets, y, cols, group, shift):
    y = y.copy()
    for e in range(w.shape[0]):
        p = np.arange(offsets[e], offsets[e + 1])
        if len(p):
            y[p] = ref_w4(w[e], scale[e], gather(x, rows_of, p, cols), cols, group, shift)
    return y


def ref_grouped(a, rows, b, offsets, scale, c, shift, bt):
    c = c.copy()
    for e in range(b.shape[0]):
        p = np.arange(offsets[e], offsets[e + 1])
        if not len(p):
            continue
        be = b[e].T if bt else b[e]
        # float64 is exact for these sums (below 2^53) and much faster than int64 @
        acc = low32((gather(a, rows, p, be.shape[0]).astype(np.float64) @ be.astype(np.float64)).astype(np.int64))
        c[p] = acc if scale is None else low32((acc.astype(np.int64) * scale[e].astype(np.int64)) >> shift)
    return c


def ref_plan(ids, experts, per, rows):
    rows, place = rows.copy(), np.full(ids.size, -1, I32)
    offsets, at = np.zeros(experts + 1, I32), 0
    for e in range(experts):
        for i in np.flatnonzero(ids == e):
            rows[at], place[i], at = i // per, at, at + 1
        offsets[e + 1] = at
    return offsets, rows, place


def sizes_to_offsets(sizes, start=0):
    return np.concatenate([[start], start + np.cumsum(sizes)]).astype(I32)


def x_of(rng, kind, shape, extreme=False):
    t = {"i8": np.int8, "i16": np.int16, "q16": np.int32}[kind]
    i = np.iinfo(t)
    if extreme:
        return rng.choice(np.array([i.min, i.min + 1, -1, 0, 1, i.max - 1, i.max], t), shape)
    return rng.integers(i.min, i.max, shape, dtype=t, endpoint=True)


def w4_of(rng, *shape):
    return rng.integers(-128, 127, shape, dtype=np.int8, endpoint=True)


def scale_of(rng, *shape):
    return rng.integers(-32768, 32767, shape, dtype=np.int16, endpoint=True)


# ------------------------------------------------------------------------ refusals (no GPU)
W, S, X, Y = np.zeros(64, np.int8), np.zeros(8, np.int16), np.zeros(64, I32), np.zeros(64, I32)
OFF = np.array([0, 1, 2], I32)


def refused(code, fn, *args):
    with pytest.raises(mind_b200.MindB200Error) as e:
        fn(*args)
    assert e.value.code == code, str(e.value)


@pytest.mark.parametrize("fn", [blas.gemv_w4_i8, blas.gemv_w4_i16, blas.gemv_w4_q16])
def test_gemv_w4_refuses(fn):
    bad = lambda *a: refused(mind_b200.ERR_INVALID, fn, *a)  # noqa: E731
    bad(W, S, X, Y, -1, 1, 32, 32, 0)
    bad(W, S, X, Y, 1, -1, 32, 32, 0)
    bad(W, S, X, Y, 1, 1, -1, 32, 0)
    bad(W, S, X, Y, 1, 1, 32, 0, 0)
    bad(W, S, X, Y, 1, 1, 32, 48, 0)
    bad(W, S, X, Y, 1, 1, 32, -32, 0)
    bad(W, S, X, Y, 1, 1, 32, 32, -1)
    bad(W, S, X, Y, 1, 1, 32, 32, 29)
    bad(0, S, X, Y, 1, 1, 32, 32, 0)
    bad(W, 0, X, Y, 1, 1, 32, 32, 0)
    bad(W, S, 0, Y, 1, 1, 32, 32, 0)
    bad(W, S, X, 0, 1, 1, 32, 32, 0)
    bad(W, S.ctypes.data + 1, X, Y, 1, 1, 32, 32, 0)
    bad(W, S, X, Y.ctypes.data + 2, 1, 1, 32, 32, 0)
    if fn is not blas.gemv_w4_i8:
        bad(W, S, X.ctypes.data + 1, Y, 1, 1, 32, 32, 0)
    refused(mind_b200.ERR_TOO_LARGE, fn, W, S, X, Y, 1, 1 << 31, 32, 32, 0)
    refused(mind_b200.ERR_TOO_LARGE, fn, W, S, X, Y, 1, 1, 1 << 31, 32, 0)
    assert fn(0, 0, 0, 0, 0, 5, 32, 32, 0) == 0  # nothing to do
    assert fn(0, 0, 0, 0, 5, 0, 32, 32, 0) == 0


def test_gemv_w4_grouped_refuses():
    fn = blas.gemv_w4_grouped_i8
    bad = lambda *a: refused(mind_b200.ERR_INVALID, fn, *a)  # noqa: E731
    bad(W, S, X, 0, 0, Y, 2, 1, 32, 32, 0, 2, 2)  # no offsets
    bad(W, S, X, 0, OFF, Y, 2, 1, 32, 32, 0, 2, 3)  # no row indices, but x has another number of rows
    bad(W, S, X, 0, OFF, Y, 2, 1, 32, 32, 0, -1, 2)
    bad(W, S, X, 0, OFF.ctypes.data + 1, Y, 2, 1, 32, 32, 0, 2, 2)
    bad(W, S, X, 0, np.array([0, 3, 2], I32), Y, 2, 1, 32, 32, 0, 2, 2)
    bad(W, S, X, 0, np.array([-1, 1, 2], I32), Y, 2, 1, 32, 32, 0, 2, 2)
    bad(W, S, X, 0, np.array([0, 1, 3], I32), Y, 2, 1, 32, 32, 0, 2, 2)
    refused(mind_b200.ERR_TOO_LARGE, fn, W, S, X, 0, OFF, Y, 2, 1, 32, 32, 0, 4097, 2)


@pytest.mark.parametrize("fn", [blas.matmul_grouped_i8, blas.matmul_grouped_i8_bt])
def test_matmul_grouped_refuses(fn):
    bad = lambda *a: refused(mind_b200.ERR_INVALID, fn, *a)  # noqa: E731
    bad(W, 0, W, OFF, 0, Y, -1, 4, 4, 2, 2)
    bad(W, 0, W, OFF, 0, Y, 2, -4, 4, 2, 2)
    bad(W, 0, W, OFF, 0, Y, 2, 4, -4, 2, 2)
    bad(W, 0, W, OFF, 0, Y, 2, 4, 4, -2, 2)
    bad(W, 0, W, OFF, 0, Y, 2, 4, 4, 2, 3)  # no row indices, but a has another number of rows
    bad(W, OFF, W, OFF, 0, Y, 2, 4, 4, 2, -1)
    bad(W, 0, W, OFF, 0, Y, 2, 4, 4, 2, 2, 63)
    bad(W, 0, W, OFF, 0, Y, 2, 4, 4, 2, 2, -1)
    bad(0, 0, W, OFF, 0, Y, 2, 4, 4, 2, 2)
    bad(W, 0, 0, OFF, 0, Y, 2, 4, 4, 2, 2)
    bad(W, 0, W, 0, 0, Y, 2, 4, 4, 2, 2)
    bad(W, 0, W, OFF, 0, 0, 2, 4, 4, 2, 2)
    bad(W, 0, W, OFF, X.ctypes.data + 2, Y, 2, 4, 4, 2, 2)
    bad(W, 0, W, OFF, 0, Y.ctypes.data + 1, 2, 4, 4, 2, 2)
    bad(W, 0, W, np.array([0, 2, 1], I32), 0, Y, 2, 4, 4, 2, 2)
    bad(W, 0, W, np.array([0, 2, 3], I32), 0, Y, 2, 4, 4, 2, 2)
    refused(mind_b200.ERR_TOO_LARGE, fn, W, 0, W, OFF, 0, Y, 2, 4, 1 << 31, 2, 2)
    refused(mind_b200.ERR_TOO_LARGE, fn, W, 0, W, OFF, 0, Y, 2, 4, 4, 4097, 2)
    assert fn(0, 0, 0, 0, 0, 0, 0, 4, 4, 2, 0) == 0
    assert fn(0, 0, 0, 0, 0, 0, 2, 4, 0, 2, 2) == 0
    assert fn(0, 0, 0, 0, 0, 0, 2, 4, 4, 0, 2) == 0


def test_expert_plan_refuses():
    bad = lambda *a: refused(mind_b200.ERR_INVALID, blas.expert_plan, *a)  # noqa: E731
    bad(X, Y, X, Y, -1, 4, 1)
    bad(X, Y, X, Y, 4, 0, 1)
    bad(X, Y, X, Y, 4, -4, 1)
    bad(X, Y, X, Y, 4, 4, 0)
    bad(0, Y, X, Y, 4, 4, 1)
    bad(X, 0, X, Y, 4, 4, 1)
    bad(X, Y, 0, Y, 4, 4, 1)
    bad(X, Y, X, 0, 4, 4, 1)
    bad(X.ctypes.data + 1, Y, X, Y, 4, 4, 1)
    refused(mind_b200.ERR_TOO_LARGE, blas.expert_plan, X, Y, X, Y, 4, 4097, 1)
    refused(mind_b200.ERR_TOO_LARGE, blas.expert_plan, X, Y, X, Y, 1 << 31, 4, 1)


def test_no_gpu_means_a_clean_refusal():
    if blas.device_count() > 0:
        pytest.skip("a B200 is present; the refusal path is for machines without one")
    refused(mind_b200.ERR_NO_DEVICE, blas.gemv_w4_q16, W, S, X, Y, 1, 1, 32, 32, 0)
    refused(mind_b200.ERR_NO_DEVICE, blas.matmul_grouped_i8, W, 0, W, OFF, 0, Y, 2, 4, 4, 2, 2)
    refused(mind_b200.ERR_NO_DEVICE, blas.expert_plan, X, Y, X, Y, 4, 4, 1)


SHIM_CHILD = r"""
import ctypes as C, sys
import numpy as np
L = C.CDLL(sys.argv[1])
i64 = C.c_int64
def fn(name, n):
    f = getattr(L, name); f.argtypes, f.restype = [i64] * n, i64
    return f
L.mind_b200_native_last_error.restype = C.c_char_p
a = np.zeros(64, np.int32); p = a.ctypes.data
names = {9: ["gemv_w4_i8", "gemv_w4_i16", "gemv_w4_q16"], 7: ["expert_plan"], 12: ["matmul_grouped_i8", "matmul_grouped_i8_bt"],
         13: ["gemv_w4_grouped_i8", "gemv_w4_grouped_i16", "gemv_w4_grouped_q16"]}
args = {9: (p, p, p, p, 1, 1, 32, 32, 99), 7: (p, p, p, p, -1, 4, 1), 12: (p, 0, p, p, 0, p, 2, 4, 4, 2, 2, 99),
        13: (p, p, p, 0, p, p, 2, 1, 32, 32, 99, 2, 2)}
for n, group in names.items():
    for name in group:
        assert fn("__mind_b200_" + name, n)(*args[n]) == int(sys.argv[2]), name
print("ok")
"""


@pytest.mark.parametrize("library,status", [(mind_b200.LIB_PATH, -1), ("/nonexistent/libmind_b200.so", -3)],
                         ids=["forwards", "missing"])
def test_native_sources_file_forwards(tmp_path, library, status):
    """integration/mind_b200_native.c resolves the new names too, and hands on the library's own checks."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    shim = str(tmp_path / "libshim.so")
    subprocess.run(["gcc", "-O2", "-Wall", "-Wextra", "-Werror", "-fPIC", "-shared", "-o", shim,
                    os.path.join(root, "integration", "mind_b200_native.c"), "-ldl", "-lpthread"], check=True)
    r = subprocess.run([sys.executable, "-c", SHIM_CHILD, shim, str(status)], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, MIND_B200_LIB=library))
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr


# ------------------------------------------------------------------------------- on a GPU
PATHS = {"default": 0, "cross-check": 1}
GROUPED_PATHS = {**PATHS, "pairs": 2, "single": 3, "square": 5, "small": 10}


@pytest.fixture(params=list(PATHS))
def path(request, gpu):
    """Both kernel families: the default one and the CUDA-core cross-check."""
    gpu.set_gemm_path(PATHS[request.param])
    yield request.param
    gpu.set_gemm_path(0)


@pytest.fixture(params=list(GROUPED_PATHS))
def grouped_path(request, gpu):
    """The grouped product's kernels: by shape, cross-check, 256 x 256 tiles on CTA pairs, 128 x 256, 128 x 128, 32 x 128."""
    gpu.set_gemm_path(GROUPED_PATHS[request.param])
    yield request.param
    gpu.set_gemm_path(0)


@pytest.fixture
def torch_gpu(gpu):
    import torch
    gpu.set_stream(torch.cuda.current_stream().cuda_stream)
    yield torch
    gpu.set_stream(0)


def dev(torch, *arrays):
    return [None if a is None else torch.from_numpy(a).cuda() for a in arrays]


@pytest.mark.gpu
@pytest.mark.parametrize("count,experts,per", [
    (0, 3, 1), (1, 1, 1), (7, 4, 1), (64, 8, 8), (33, 33, 3), (1000, 5, 2), (1024, 256, 8), (4097, 160, 6), (65536, 64, 8),
    (70001, 3, 7), (5000, 4096, 2), (300000, 512, 4)])
def test_expert_plan(gpu, count, experts, per):
    rng = np.random.default_rng(count * 31 + experts)
    for padding in (0.0, 0.3, 1.0):
        ids = rng.integers(0, experts, count, dtype=I32)
        bad = rng.random(count) < padding
        ids[bad] = rng.choice(np.array([-1, -(2 ** 31), experts, 2 ** 31 - 1], I32), int(bad.sum()))
        rows, place, offsets = (np.full(n + 5, CANARY, I32) for n in (count, count, experts + 1))
        want = ref_plan(ids, experts, per, rows)
        gpu.expert_plan(ids, offsets, rows, place, count, experts, per)
        assert np.array_equal(offsets[:experts + 1], want[0])
        assert np.array_equal(rows, want[1])  # what lies behind the kept slots is as it was
        assert np.array_equal(place[:count], want[2])
        assert np.all(place[count:] == CANARY) and np.all(offsets[experts + 1:] == CANARY)


@pytest.mark.gpu
def test_expert_plan_one_popular_expert(gpu):
    """Every slot of one expert, and experts in descending order."""
    for ids in (np.full(20000, 6, I32), np.repeat(np.arange(49, -1, -1), 37).astype(I32)):
        offsets, rows, place = np.zeros(51, I32), np.zeros(ids.size, I32), np.zeros(ids.size, I32)
        gpu.expert_plan(ids, offsets, rows, place, ids.size, 50, 1)
        want = ref_plan(ids, 50, 1, rows)
        for got, expected in zip((offsets, rows, place), want):
            assert np.array_equal(got, expected)


# Block edges of the kernels: 16 rows, 32 / 256 columns, 8 tokens; odd columns (a half-filled last byte).
W4_SHAPES = [
    (1, 1, 1, 32), (1, 1, 32, 32), (1, 16, 256, 64), (2, 17, 255, 128), (3, 33, 257, 32), (8, 48, 512, 256),
    (9, 15, 96, 96), (5, 100, 1000, 64), (4, 64, 2048, 128), (7, 31, 777, 1024), (16, 40, 1056, 32), (17, 129, 640, 160),
    (32, 65, 800, 128), (33, 20, 320, 64), (70, 18, 416, 32), (1, 300, 4096, 128), (2, 2500, 1024, 512), (3, 1030, 544, 32),
    (1, 16, 20000, 128), (8, 24, 9000, 64), (6, 40, 0, 32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["i8", "i16", "q16"])
def test_gemv_w4_shapes(gpu, path, kind):
    fn = getattr(gpu, f"gemv_w4_{kind}")
    for (t, rows, cols, group) in W4_SHAPES:
        rng = np.random.default_rng(t * 1000003 + rows * 1009 + cols)
        groups = -(-cols // group)
        w, s, x = w4_of(rng, rows, (cols + 1) // 2), scale_of(rng, rows, groups), x_of(rng, kind, (t, cols))
        for shift in (0, 11, 28):
            y = np.full(t * rows + 8, CANARY, I32)
            fn(w, s, x, y, t, rows, cols, group, shift)
            want = ref_w4(w, s, x, cols, group, shift)
            assert np.array_equal(y[:t * rows].reshape(t, rows), want), (t, rows, cols, group, shift)
            assert np.all(y[t * rows:] == CANARY)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["i8", "i16", "q16"])
def test_gemv_w4_extreme_values(gpu, path, kind):
    """The ends of every type, all at once and mixed: nothing saturates, every limb carries."""
    rng = np.random.default_rng(5)
    i = np.iinfo({"i8": np.int8, "i16": np.int16, "q16": np.int32}[kind])
    for (t, rows, cols, group) in [(1, 32, 4096, 4096), (8, 16, 1024, 1024), (2, 16, 8192, 32), (3, 50, 333, 64)]:
        groups = -(-cols // group)
        cases = [(np.full((rows, (cols + 1) // 2), -120, np.int8), v, m) for v in (i.min, i.max) for m in (-32768, 32767)]
        cases += [(w4_of(rng, rows, (cols + 1) // 2), None, None)]
        for w, v, m in cases:
            x = x_of(rng, kind, (t, cols), extreme=True) if v is None else np.full((t, cols), v, dtype=i.dtype)
            s = scale_of(rng, rows, groups) if m is None else np.full((rows, groups), m, np.int16)
            for shift in (0, 20, 28):
                y = np.empty((t, rows), I32)
                getattr(gpu, f"gemv_w4_{kind}")(w, s, x, y, t, rows, cols, group, shift)
                assert np.array_equal(y, ref_w4(w, s, x, cols, group, shift)), (t, rows, cols, shift, v, m)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["i8", "i16", "q16"])
def test_gemv_w4_odd_bases(torch_gpu, gpu, path, kind):
    """Device operands whose bases are aligned to their element alone."""
    torch = torch_gpu
    rng = np.random.default_rng(9)
    for (t, rows, cols, group) in [(1, 40, 512, 128), (5, 33, 1024, 32)]:
        w, s, x = w4_of(rng, rows, cols // 2), scale_of(rng, rows, cols // group), x_of(rng, kind, (t, cols))
        want = ref_w4(w, s, x, cols, group, 9)

        def shifted(a, by=1):
            base = torch.zeros(a.size + by, dtype=torch.from_numpy(a).dtype, device="cuda")
            base[by:] = torch.from_numpy(a.reshape(-1)).cuda()
            return base[by:]

        y = torch.full((t * rows + 3,), CANARY, dtype=torch.int32, device="cuda")
        getattr(gpu, f"gemv_w4_{kind}")(shifted(w, 3), shifted(s), shifted(x), y[1:], t, rows, cols, group, 9)
        got = y.cpu().numpy()
        assert np.array_equal(got[1:1 + t * rows].reshape(t, rows), want)
        assert got[0] == CANARY and np.all(got[1 + t * rows:] == CANARY)


GROUP_SIZES = [[1], [5, 0, 3], [0, 0, 7, 0], [16, 17, 1, 40], [0], [9, 33, 64, 2, 0, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["i8", "i16", "q16"])
@pytest.mark.parametrize("sizes", GROUP_SIZES, ids=str)
def test_gemv_w4_grouped(gpu, path, kind, sizes):
    rng = np.random.default_rng(len(sizes) * 7 + sum(sizes))
    fn = getattr(gpu, f"gemv_w4_grouped_{kind}")
    for (rows, cols, group) in [(35, 320, 32), (64, 1024, 128), (19, 201, 64)]:
        experts, groups = len(sizes), -(-cols // group)
        offsets = sizes_to_offsets(sizes, start=2)  # two rows before the first group, three behind the last
        m, x_rows = int(offsets[-1]) + 3, 11
        w, s = w4_of(rng, experts, rows, (cols + 1) // 2), scale_of(rng, experts, rows, groups)
        x = x_of(rng, kind, (x_rows, cols))
        rows_of = rng.integers(0, x_rows, m).astype(I32)
        rows_of[rng.random(m) < 0.1] = rng.choice([-1, x_rows, 2 ** 31 - 1])  # such a row counts as zeros
        y0 = rng.integers(-9, 9, (m, rows)).astype(I32)
        y = y0.copy()
        fn(w, s, x, rows_of, offsets, y, m, rows, cols, group, 7, experts, x_rows)
        assert np.array_equal(y, ref_w4_grouped(w, s, x, rows_of, offsets, y0, cols, group, 7)), (rows, cols)
        xm, y = x_of(rng, kind, (m, cols)), y0.copy()
        fn(w, s, xm, None, offsets, y, m, rows, cols, group, 7, experts, m)
        assert np.array_equal(y, ref_w4_grouped(w, s, xm, None, offsets, y0, cols, group, 7)), (rows, cols)


# Tile edges of the grouped kernels: 32 / 128 / 256 rows, 64 / 128 / 256 columns, 128 of K, 16-byte pitches.
GROUPED_SHAPES = [
    ([1], 16, 16), ([3, 0, 130], 128, 64), ([129, 257, 1], 144, 272), ([0, 0, 31], 1, 1), ([40, 41], 129, 130),
    ([300, 5, 0, 64], 256, 256), ([7] * 20, 400, 48), ([500, 20], 96, 528), ([2, 2, 2], 33, 20), ([256, 128], 1040, 128),
    ([12, 0, 9], 0, 40),
]


@pytest.mark.gpu
@pytest.mark.parametrize("bt", [False, True], ids=["kn", "nk"])
@pytest.mark.parametrize("sizes,k,n", GROUPED_SHAPES, ids=str)
def test_matmul_grouped_shapes(gpu, grouped_path, bt, sizes, k, n):
    rng = np.random.default_rng(sum(sizes) + k * 7 + n)
    experts = len(sizes)
    fn = gpu.matmul_grouped_i8_bt if bt else gpu.matmul_grouped_i8
    offsets = sizes_to_offsets(sizes, start=3)
    m, a_rows = int(offsets[-1]) + 2, 50
    b = rng.integers(-128, 127, (experts, n, k) if bt else (experts, k, n), dtype=np.int8, endpoint=True)
    scale = rng.integers(-(2 ** 31), 2 ** 31 - 1, (experts, n), dtype=I32, endpoint=True)
    c0 = rng.integers(-9, 9, (m, n)).astype(I32)
    rows = rng.integers(0, a_rows, m).astype(I32)
    rows[rng.random(m) < 0.1] = rng.choice([-1, a_rows, 2 ** 31 - 1])
    for ri in (rows, None):
        a = rng.integers(-128, 127, (a_rows if ri is not None else m, k), dtype=np.int8, endpoint=True)
        for sc, shift in ((None, 0), (scale, 0), (scale, 31), (scale, 62)):
            c = c0.copy()
            fn(a, ri, b, offsets, sc, c, m, k, n, experts, a.shape[0], shift)
            assert np.array_equal(c, ref_grouped(a, ri, b, offsets, sc, c0, shift, bt)), (ri is not None, shift)


@pytest.mark.gpu
def test_matmul_grouped_wraps(gpu, grouped_path):
    """Sums past 2^31 wrap (K * 2^14 with K = 2^17 + 256), with and without a scale."""
    k = (1 << 17) + 256
    a, b = np.full((3, k), -128, np.int8), np.full((2, k, 16), -128, np.int8)
    offsets, scale = np.array([0, 1, 3], I32), np.full((2, 16), -3, I32)
    want = low32(np.full((3, 16), k << 14, np.int64))
    for sc in (None, scale):
        c = np.zeros((3, 16), I32)
        gpu.matmul_grouped_i8(a, None, b, offsets, sc, c, 3, k, 16, 2, 3, 1)
        assert np.array_equal(c, want if sc is None else low32((want.astype(np.int64) * -3) >> 1))


@pytest.mark.gpu
@pytest.mark.parametrize("bt", [False, True], ids=["kn", "nk"])
def test_matmul_grouped_device_operands(torch_gpu, gpu, grouped_path, bt):
    """Device operands, aligned and not, on sizes where whole and partial tiles meet."""
    torch = torch_gpu
    rng = np.random.default_rng(21)
    fn = gpu.matmul_grouped_i8_bt if bt else gpu.matmul_grouped_i8
    sizes, k, n = [700, 0, 33, 1, 260], 384, 320
    offsets = sizes_to_offsets(sizes)
    m = int(offsets[-1])
    a = rng.integers(-128, 127, (m, k), dtype=np.int8, endpoint=True)
    b = rng.integers(-128, 127, (5, n, k) if bt else (5, k, n), dtype=np.int8, endpoint=True)
    want = ref_grouped(a, None, b, offsets, None, np.zeros((m, n), I32), 0, bt)
    for by_a, by_b, by_c in ((0, 0, 0), (1, 0, 0), (0, 3, 0), (0, 0, 1), (5, 16, 2)):
        da, db = torch.zeros(a.size + by_a, dtype=torch.int8, device="cuda"), torch.zeros(b.size + by_b, dtype=torch.int8, device="cuda")
        da[by_a:], db[by_b:] = torch.from_numpy(a.reshape(-1)).cuda(), torch.from_numpy(b.reshape(-1)).cuda()
        c = torch.full((m * n + by_c + 4,), CANARY, dtype=torch.int32, device="cuda")
        fn(da[by_a:], None, db[by_b:], torch.from_numpy(offsets).cuda(), None, c[by_c:], m, k, n, 5, m)
        got = c.cpu().numpy()
        assert np.array_equal(got[by_c:by_c + m * n].reshape(m, n), want), (by_a, by_b, by_c)
        assert np.all(got[:by_c] == CANARY) and np.all(got[by_c + m * n:] == CANARY)


@pytest.mark.gpu
def test_wrong_device_offsets_stay_inside(torch_gpu, gpu, grouped_path):
    """Offsets in device memory cannot be refused; the kernels take each bound no lower than the one before
    and no higher than m, so nothing outside the output is written."""
    torch = torch_gpu
    rng = np.random.default_rng(3)
    m, k, n, rows = 40, 64, 48, 20
    a, b = rng.integers(-9, 9, (m, k)).astype(np.int8), rng.integers(-9, 9, (3, k, n)).astype(np.int8)
    w, s = w4_of(rng, 3, rows, k // 2), scale_of(rng, 3, rows, 2)
    for off in ([0, 50, 20, 45], [-7, 10, 2 ** 31 - 1, 3], [60, 70, 80, 90], [0, 0, 0, 0], [30, 20, 10, 0]):
        da, db, dw, ds, do = dev(torch, a, b, w, s, np.array(off, I32))
        c = torch.full((m * n + 64,), CANARY, dtype=torch.int32, device="cuda")
        y = torch.full((m * rows + 64,), CANARY, dtype=torch.int32, device="cuda")
        gpu.matmul_grouped_i8(da, None, db, do, None, c, m, k, n, 3, m)
        gpu.gemv_w4_grouped_i8(dw, ds, da, None, do, y, m, rows, k, 32, 0, 3, m)
        gpu.synchronize()
        assert np.all(c.cpu().numpy()[m * n:] == CANARY) and np.all(y.cpu().numpy()[m * rows:] == CANARY)
        bounds, before = [], 0
        for v in off:
            before = min(max(v, before), m)
            bounds.append(before)
        want = ref_grouped(a, None, b, np.array(bounds, I32), None, np.full((m, n), CANARY, I32), 0, False)
        assert np.array_equal(c.cpu().numpy()[:m * n].reshape(m, n), want), off
        want = ref_w4_grouped(w, s, a, None, np.array(bounds, I32), np.full((m, rows), CANARY, I32), k, 32, 0)
        assert np.array_equal(y.cpu().numpy()[:m * rows].reshape(m, rows), want), off


def expert_layer(gpu, torch, rng, tokens, per, experts, k, n):
    """One layer's operands on the device, and what its calls should give."""
    ids = np.stack([rng.permutation(experts)[:per] for _ in range(tokens)]).astype(I32)
    ids[tokens - tokens // 5:] = -1  # a padded batch
    x = rng.integers(-128, 127, (tokens, k), dtype=np.int8, endpoint=True)
    b = rng.integers(-128, 127, (experts, k, n), dtype=np.int8, endpoint=True)
    scale = rng.integers(0, 4000, (experts, n)).astype(I32)
    w, s = w4_of(rng, experts, k, (n + 1) // 2), scale_of(rng, experts, k, -(-n // 64))
    m = tokens * per
    offsets, rows, place = ref_plan(ids.reshape(-1), experts, per, np.full(m, CANARY, I32))
    h = ref_grouped(x, rows, b, offsets, scale, np.full((m, n), CANARY, I32), 6, False)
    y = ref_w4_grouped(w, s, h, None, offsets, np.full((m, k), CANARY, I32), n, 64, 20)
    d = dict(zip(("ids", "x", "b", "scale", "w", "s"), dev(torch, ids.reshape(-1), x, b, scale, w, s)))
    for name, size in (("offsets", experts + 1), ("rows", m), ("place", m), ("h", m * n), ("y", m * k)):
        d[name] = torch.full((size,), CANARY, dtype=torch.int32, device="cuda")

    def run():
        gpu.expert_plan(d["ids"], d["offsets"], d["rows"], d["place"], m, experts, per)
        gpu.matmul_grouped_i8(d["x"], d["rows"], d["b"], d["offsets"], d["scale"], d["h"], m, k, n, experts, tokens, 6)
        gpu.gemv_w4_grouped_q16(d["w"], d["s"], d["h"], None, d["offsets"], d["y"], m, k, n, 64, 20, experts, m)

    def check():
        torch.cuda.synchronize()
        for name, want in (("offsets", offsets), ("rows", rows), ("place", place), ("h", h), ("y", y)):
            assert np.array_equal(d[name].cpu().numpy(), want.reshape(-1)), name

    return d, run, check


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,per,experts,k,n", [(1, 2, 4, 64, 96), (6, 2, 8, 128, 160), (40, 3, 16, 256, 384),
                                                    (150, 2, 5, 200, 133)])
def test_expert_layer(torch_gpu, gpu, path, tokens, per, experts, k, n):
    """Plan, grouped product, 4-bit product, each fed by the one before, on a padded batch."""
    _, run, check = expert_layer(gpu, torch_gpu, np.random.default_rng(tokens), tokens, per, experts, k, n)
    for _ in range(3):
        run()
    check()


@pytest.mark.gpu
def test_expert_layer_captured_and_replayed(torch_gpu, gpu):
    """The layer captured on a side stream and replayed on new tokens: sizes of groups are read on the device."""
    torch = torch_gpu
    rng = np.random.default_rng(4)
    d, run, _ = expert_layer(gpu, torch, rng, 24, 2, 6, 192, 128)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        gpu.set_stream(stream.cuda_stream)
        run()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run()
    for seed in (5, 6):
        d2, _, _ = expert_layer(gpu, torch, np.random.default_rng(seed), 24, 2, 6, 192, 128)
        for name in d:
            d[name].copy_(d2[name])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ids = d["ids"].cpu().numpy()
        offsets, rows, place = ref_plan(ids, 6, 2, np.full(48, CANARY, I32))
        h = ref_grouped(d["x"].cpu().numpy(), rows, d["b"].cpu().numpy(), offsets, d["scale"].cpu().numpy(),
                        np.full((48, 128), CANARY, I32), 6, False)
        y = ref_w4_grouped(d["w"].cpu().numpy(), d["s"].cpu().numpy(), h, None, offsets, np.full((48, 192), CANARY, I32),
                           128, 64, 20)
        for name, want in (("offsets", offsets), ("rows", rows), ("place", place), ("h", h), ("y", y)):
            assert np.array_equal(d[name].cpu().numpy(), want.reshape(-1)), name
    gpu.set_stream(0)


@pytest.mark.gpu
def test_two_threads_at_once(torch_gpu, gpu):
    torch = torch_gpu
    layers = [expert_layer(gpu, torch, np.random.default_rng(s), 30, 2, 6, 160, 224) for s in (1, 2)]
    errors = []

    def work(run):
        try:
            for _ in range(20):
                run()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(layer[1],)) for layer in layers]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for layer in layers:
        layer[2]()


@pytest.mark.gpu
def test_same_bytes_every_time(torch_gpu, gpu):
    torch = torch_gpu
    d, run, check = expert_layer(gpu, torch, np.random.default_rng(8), 64, 4, 8, 256, 512)
    run()
    check()
    first = {n: d[n].clone() for n in ("h", "y")}
    for _ in range(50):
        for n in first:
            d[n].fill_(CANARY)
        run()
        for n, v in first.items():
            assert torch.equal(d[n], v)


@pytest.mark.gpu
def test_operands_of_another_device_are_refused(torch_gpu, gpu):
    torch = torch_gpu
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    y = torch.zeros(16, dtype=torch.int32, device="cuda:1")
    z = torch.zeros(64, dtype=torch.int8, device="cuda:0")
    refused(mind_b200.ERR_INVALID, gpu.gemv_w4_i8, z, z, z, y, 1, 1, 32, 32, 0)


@pytest.mark.gpu
def test_weights_past_32_bits(torch_gpu, gpu):
    """Stacks of weights of more than 2^31 bytes, and an output of more than 2^31 elements."""
    torch = torch_gpu
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    i32 = dict(dtype=torch.int32, device="cuda")

    def some(shape, dtype=torch.int8):
        return torch.randint(-128, 128, shape, generator=gen, device="cuda", dtype=torch.int16).to(dtype)

    # 4-bit: 70 experts of 4096 x 16384
    experts, rows, cols, group = 70, 4096, 16384, 128
    w, s, x = some((experts, rows, cols // 2)), some((experts, rows, cols // group), torch.int16), some((3, cols))
    assert w.numel() > 2 ** 31
    offsets = torch.zeros(experts + 1, **i32)
    offsets[1:] = 1
    offsets[-1] = 3
    y = torch.zeros((3, rows), **i32)
    gpu.gemv_w4_grouped_i8(w, s, x, None, offsets, y, 3, rows, cols, group, 8, experts, 3)
    got = y.cpu().numpy()
    for p, e in ((0, 0), (1, experts - 1), (2, experts - 1)):
        want = ref_w4(w[e].cpu().numpy(), s[e].cpu().numpy(), x[p:p + 1].cpu().numpy(), cols, group, 8)
        assert np.array_equal(got[p:p + 1], want), p
    del w

    # int8: nine experts of 16384 x 16384, both orientations
    experts, k, n = 9, 16384, 16384
    b, a = some((experts, k, n)), some((40, k))
    assert b.numel() > 2 ** 31
    offsets = torch.full((experts + 1,), 7, **i32)
    offsets[0] = 0
    offsets[-1] = 40
    c = torch.zeros((40, n), **i32)
    for bt, fn in ((False, gpu.matmul_grouped_i8), (True, gpu.matmul_grouped_i8_bt)):
        fn(a, None, b, offsets, None, c, 40, k, n, experts, 40)
        for lo, hi, e in ((0, 7, 0), (7, 40, experts - 1)):
            part = b[e, -96:].t() if bt else b[e, :, -96:]
            want = torch.matmul(a[lo:hi].double(), part.double()).long().to(torch.int32)
            assert torch.equal(c[lo:hi, -96:], want), (bt, e)
    del b, c

    # an output of 2.2e9 elements
    m, k, n = 68000, 32, 32256
    a, b = some((m, k)), some((2, k, n))
    offsets = torch.tensor([0, 30001, m], **i32)
    c = torch.zeros((m, n), **i32)
    assert c.numel() > 2 ** 31
    gpu.matmul_grouped_i8(a, None, b, offsets, None, c, m, k, n, 2, m)
    for lo, hi, e in ((0, 5, 0), (29990, 30001, 0), (30001, 30010, 1), (m - 9, m, 1)):
        want = torch.matmul(a[lo:hi].double(), b[e].double()).long().to(torch.int32)
        assert torch.equal(c[lo:hi], want), (lo, e)


@pytest.mark.gpu
@pytest.mark.parametrize("count,experts", [(16384, 17), (16385, 17), (3_000_000, 384), (2_000_000, 2500)])
def test_expert_plan_large(torch_gpu, gpu, count, experts):
    """Both forms at their border, and long batches, against a stable sort."""
    torch = torch_gpu
    gen = torch.Generator(device="cuda")
    gen.manual_seed(count)
    ids = torch.randint(-1, experts, (count,), generator=gen, device="cuda", dtype=torch.int32)
    offsets, rows, place = (torch.full((n,), CANARY, dtype=torch.int32, device="cuda") for n in (experts + 1, count, count))
    gpu.expert_plan(ids, offsets, rows, place, count, experts, 3)
    key = torch.where(ids >= 0, ids, experts).long()
    order = torch.sort(key, stable=True).indices
    kept = int((ids >= 0).sum())
    assert torch.equal(offsets.long(), torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"),
                                                  torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0)]))
    assert torch.equal(rows[:kept].long(), order[:kept] // 3) and bool((rows[kept:] == CANARY).all())
    want = torch.full((count,), -1, dtype=torch.int32, device="cuda")
    want[order[:kept]] = torch.arange(kept, dtype=torch.int32, device="cuda")
    assert torch.equal(place, want)


@pytest.mark.gpu
def test_two_graphs_one_after_the_other(torch_gpu, gpu):
    """Two captured layers that share the library's scratch (gathered rows, odd columns), replayed in turn and
    mixed with eager calls of a third."""
    torch = torch_gpu
    layers = [expert_layer(gpu, torch, np.random.default_rng(s), 50, 2, 5, 130 + s, 95) for s in (1, 2, 3)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        gpu.set_stream(stream.cuda_stream)
        for _, run, _ in layers:
            run()
        stream.synchronize()
        for _, run, _ in layers[:2]:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                run()
            graphs.append(graph)
        for d, _, _ in layers:
            for name in ("offsets", "rows", "place", "h", "y"):
                d[name].fill_(CANARY)
        for _ in range(3):
            graphs[0].replay()
            layers[2][1]()
            graphs[1].replay()
        stream.synchronize()
    for layer in layers:
        layer[2]()
    gpu.set_stream(0)


@pytest.mark.gpu
def test_other_streams(torch_gpu, gpu):
    """Each call's operands are made on the stream it runs on, without a wait in between."""
    torch = torch_gpu
    layers = []
    for s in (1, 2):
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            gpu.set_stream(stream.cuda_stream)
            layer = expert_layer(gpu, torch, np.random.default_rng(s), 60, 2, 6, 256, 320)
            for name in ("x", "w", "s"):  # queued on the same stream right before the calls
                layer[0][name].add_(1).sub_(1)
            layer[1]()
            layers.append(layer)
    for layer in layers:
        layer[2]()


@pytest.mark.gpu
def test_pinned_offsets_written_in_stream_order(torch_gpu, gpu):
    """Offsets in pinned memory may still be on their way when the call is made: they are not looked at then."""
    torch = torch_gpu
    rng = np.random.default_rng(9)
    m, k, n, experts = 20, 64, 48, 3
    a, b = rng.integers(-128, 128, (m, k), dtype=np.int8), rng.integers(-128, 128, (experts, k, n), dtype=np.int8)
    offsets = np.array([0, 6, 6, m], dtype=np.int32)
    da, db, do = dev(torch, a, b, offsets)
    pinned = torch.full((experts + 1,), CANARY, dtype=torch.int32).pin_memory()
    c = torch.full((m, n), CANARY, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    gpu.set_stream(stream.cuda_stream)
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        pinned.copy_(do, non_blocking=True)
        gpu.matmul_grouped_i8(da, None, db, pinned, None, c, m, k, n, experts, m)
    gpu.set_stream(0)
    want = ref_grouped(a, None, b, offsets, None, np.full((m, n), CANARY, np.int32), 0, False)
    assert np.array_equal(c.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("experts", [1, 2, 63, 64, 255, 1025, 4096])
@pytest.mark.parametrize("count", [31, 128, 129, 256, 257, 512, 513, 1025, 2047, 2049, 8192, 8193, 16384, 16385, 40007])
def test_expert_plan_borders(gpu, count, experts):
    """Where the kernel takes another block, more warps or a second launch; few and many ids of one expert."""
    rng = np.random.default_rng(count + 100003 * experts)
    any_id = rng.integers(-1, experts + 1, count, dtype=I32)
    runs = np.sort(rng.integers(0, experts, count, dtype=I32))[::-1].copy()
    for ids in (any_id, runs, np.full(count, experts - 1, I32), np.full(count, experts, I32)):
        offsets, rows, place = (np.full(n, CANARY, I32) for n in (experts + 1, count, count))
        want = ref_plan(ids, experts, 2, rows)
        gpu.expert_plan(ids, offsets, rows, place, count, experts, 2)
        for got, expected in zip((offsets, rows, place), want):
            assert np.array_equal(got, expected)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,tokens,rows,cols,group,sets", [
    ("i8", 1, 28672, 8192, 128, 2), ("q16", 8, 16384, 8192, 32, 3), ("q16", 8, 16384, 8192, 128, 3),
    ("i16", 5, 12289, 5120, 64, 5), ("i8", 32, 8192, 8192, 256, 5)])
def test_gemv_w4_slots_are_refilled_behind_their_readers(torch_gpu, gpu, kind, tokens, rows, cols, group, sets):
    """Weights that come from memory every time (matrices larger than L2 together, taken in turn): the warps wait
    for the boxes of their ring and refill each slot as soon as it has been multiplied."""
    torch = torch_gpu
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows + group)

    def some(shape, lo, hi, dtype):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=torch.int64).to(dtype)

    lim = {"i8": 2 ** 7, "i16": 2 ** 15, "q16": 2 ** 31}[kind]
    x = some((tokens, cols), -lim, lim, {"i8": torch.int8, "i16": torch.int16, "q16": torch.int32}[kind])
    w = [torch.randint(-128, 128, (rows, cols // 2), generator=gen, device="cuda", dtype=torch.int16).to(torch.int8)
         for _ in range(sets)]
    s = [some((rows, cols // group), -2 ** 15, 2 ** 15, torch.int16) for _ in range(sets)]
    assert sets * w[0].numel() > 150_000_000  # 126 MB of L2
    fn = getattr(gpu, f"gemv_w4_{kind}")
    want = [torch.empty((tokens, rows), dtype=torch.int32, device="cuda") for _ in range(sets)]
    gpu.set_gemm_path(1)
    for i in range(sets):
        fn(w[i], s[i], x, want[i], tokens, rows, cols, group, 9)
    gpu.set_gemm_path(0)
    y = torch.empty((tokens, rows), dtype=torch.int32, device="cuda")
    wrong = torch.zeros(1, dtype=torch.int64, device="cuda")
    for n in range(40 * sets):
        y.fill_(CANARY)
        fn(w[n % sets], s[n % sets], x, y, tokens, rows, cols, group, 9)
        wrong += (y != want[n % sets]).sum()
    gpu.synchronize()
    assert int(wrong) == 0


# ------------------------------------------------------- shapes of the 4-bit kernel, asked for by name
@pytest.fixture
def w4_shape():
    yield blas.set_w4_shape
    blas.set_w4_shape()


def test_w4_shape_refuses(w4_shape):
    for bad in ((3, 0, 0), (16, 0, 0), (-1, 0, 0), (0, 17, 0), (0, -1, 0), (0, 0, 33), (0, 0, -1)):
        refused(mind_b200.ERR_INVALID, w4_shape, *bad)
    for bad in ((3, 1, 1, 32, 32), (0, 0, 1, 32, 32), (0, 1, 0, 32, 32), (0, 1, 1, 0, 32), (0, 1, 1, 32, 48), (0, 1, 1, 32, 32, -1)):
        refused(mind_b200.ERR_INVALID, blas.w4_shape, *bad)
    refused(mind_b200.ERR_TOO_LARGE, blas.w4_shape, 0, 1, 1, 32, 32, 4097)
    refused(mind_b200.ERR_TOO_LARGE, blas.w4_shape, 0, 1, 1 << 31, 32, 32)


def test_w4_shape_is_what_was_asked_for(w4_shape):
    for kind in (blas.KIND_I8, blas.KIND_I16, blas.KIND_Q16):
        for experts in (0, 8):
            free = blas.w4_shape(kind, 24, 5000, 4608, 128, experts)
            assert free["cluster"] in (1, 2, 4, 8) and 1 <= free["row_tiles"] <= 16 and 2 <= free["slots"] <= 8
            for cs, rt, tb in ((1, 5, 2), (2, 16, 0), (4, 0, 3), (8, 1, 1)):
                w4_shape(cs, rt, tb)
                got = blas.w4_shape(kind, 24, 5000, 4608, 128, experts)
                assert got["cluster"] == cs and got["row_tiles"] == (rt or got["row_tiles"])
                assert got["tokens"] == (tb or got["tokens"]) and got["rounds"] >= got["clusters"] >= 1
            w4_shape()
            assert blas.w4_shape(kind, 24, 5000, 4608, 128, experts) == free
    w4_shape(8, 0, 0)  # fewer than eight units of 512 columns
    assert blas.w4_shape(blas.KIND_I8, 1, 100, 1024, 32)["cluster"] == 0


@pytest.mark.gpu
def test_a_shape_that_does_not_fit_is_refused(gpu, w4_shape):
    w, s, x, y = np.zeros((16, 512), np.int8), np.zeros((16, 32), np.int16), np.zeros(1024, np.int8), np.zeros(16, I32)
    w4_shape(8, 0, 0)
    refused(mind_b200.ERR_INVALID, gpu.gemv_w4_i8, w, s, x, y, 1, 16, 1024, 32, 0)
    w4_shape()
    assert gpu.gemv_w4_i8(w, s, x, y, 1, 16, 1024, 32, 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["i8", "i16", "q16"])
@pytest.mark.parametrize("cs", [1, 2, 4, 8])
@pytest.mark.parametrize("rt", [1, 3, 5, 6, 16])
def test_gemv_w4_rounds(torch_gpu, gpu, w4_shape, kind, cs, rt):
    """Every cluster size and several row tiles with three or more rounds to a cluster: the ring and the sums are
    carried from one round to the next, activations change in between.  Against the cross-check kernel, and some rows
    against numpy.  Odd rows; odd columns (rows that have to be laid out) and whole ones; one matrix and grouped rows."""
    torch = torch_gpu
    gen = torch.Generator(device="cuda")
    gen.manual_seed(cs * 100 + rt)

    def some(shape, bits, dtype):
        return torch.randint(-2 ** (bits - 1), 2 ** (bits - 1), shape, generator=gen, device="cuda", dtype=torch.int64).to(dtype)

    bits, dtype = {"i8": (8, torch.int8), "i16": (16, torch.int16), "q16": (32, torch.int32)}[kind]
    code = {"i8": blas.KIND_I8, "i16": blas.KIND_I16, "q16": blas.KIND_Q16}[kind]
    # tokens whose activations fit beside the ring
    wide = {"i8": 12, "i16": 4 if cs == 1 else 12, "q16": {1: 4, 2: 7}.get(cs, 12)}[kind]
    for tb, cols, group, experts in ((1, 4608, 128, 0), (wide, 4389, 32, 0), (3, 4096 + 160, 64, 0), (2, 4100, 96, 4), (wide, 4608, 32, 4)):
        blocks = 6
        row_rounds = 3 * (148 // cs) // blocks + 1
        rows = 16 * rt * row_rounds - 5
        m = blocks * tb
        stack, groups = (experts or 1, rows), -(-cols // group)
        w = torch.randint(-128, 128, (*stack, (cols + 1) // 2), generator=gen, device="cuda", dtype=torch.int16).to(torch.int8)
        s, x = some((*stack, groups), 16, torch.int16), some((m, cols), bits, dtype)
        y, want = (torch.full((m, rows), CANARY, dtype=torch.int32, device="cuda") for _ in range(2))
        if experts:  # sizes that fill some blocks of tokens and not others
            offsets = torch.tensor([0, m // 2 + 1, m // 2 + 1, m - 1, m], dtype=torch.int32, device="cuda")
            rows_of = torch.randint(-1, m + 1, (m,), generator=gen, device="cuda", dtype=torch.int32)

        def call(out):
            if experts:
                getattr(gpu, f"gemv_w4_grouped_{kind}")(w, s, x, rows_of, offsets, out, m, rows, cols, group, 13, experts, m)
            else:
                getattr(gpu, f"gemv_w4_{kind}")(w, s, x, out, m, rows, cols, group, 13)

        gpu.set_gemm_path(1)
        call(want)
        gpu.set_gemm_path(0)
        w4_shape(cs, rt, tb)
        shape = gpu.w4_shape(code, m, rows, cols, group, experts)
        assert shape["cluster"] == cs and shape["row_tiles"] == rt and shape["rounds"] >= 3 * shape["clusters"], shape
        call(y)
        w4_shape()
        call_differs = int((y != want).sum())
        assert call_differs == 0, (tb, cols, group, experts, call_differs)
        r = np.unique(np.concatenate([[0, rows - 1], np.random.default_rng(rt).integers(0, rows, 6)]))
        xs = x.cpu().numpy()
        for e in range(experts or 1):
            lo, hi = (int(offsets[e]), int(offsets[e + 1])) if experts else (0, m)
            if hi > lo:
                xe = gather(xs, rows_of.cpu().numpy(), np.arange(lo, hi), cols) if experts else xs
                assert np.array_equal(y[lo:hi].cpu().numpy()[:, r], ref_w4(w[e].cpu().numpy()[r], s[e].cpu().numpy()[r], xe, cols, group, 13))


@pytest.mark.gpu
@pytest.mark.parametrize("kind,m,rows,cols,group", [("i8", 300, 4100, 4097, 128), ("q16", 70, 8192, 8192, 32), ("i16", 41, 20000, 5120, 64)])
def test_gemv_w4_many_tokens_by_the_estimate(torch_gpu, gpu, kind, m, rows, cols, group):
    """Shapes of several rounds that the kernel takes of its own accord."""
    torch = torch_gpu
    rng = np.random.default_rng(m)
    code = {"i8": blas.KIND_I8, "i16": blas.KIND_I16, "q16": blas.KIND_Q16}[kind]
    shape = gpu.w4_shape(code, m, rows, cols, group)
    assert shape["rounds"] > shape["clusters"], shape
    w, s, x = w4_of(rng, rows, (cols + 1) // 2), scale_of(rng, rows, -(-cols // group)), x_of(rng, kind, (m, cols))
    dw, ds, dx = dev(torch, w, s, x)
    y, want = (torch.full((m, rows), CANARY, dtype=torch.int32, device="cuda") for _ in range(2))
    fn = getattr(gpu, f"gemv_w4_{kind}")
    gpu.set_gemm_path(1)
    fn(dw, ds, dx, want, m, rows, cols, group, 5)
    gpu.set_gemm_path(0)
    for _ in range(3):
        y.fill_(CANARY)
        fn(dw, ds, dx, y, m, rows, cols, group, 5)
        assert torch.equal(y, want)
    r = rng.integers(0, rows, 8)
    assert np.array_equal(y.cpu().numpy()[:, r], ref_w4(w[r], s[r], x, cols, group, 5))


def test_w4_shape_is_found_in_a_few_tries():
    """The host's search must not grow with the number of tokens: it runs inside the call, under the device's lock."""
    for m in (1, 33, 4097, 1_000_000, 2 ** 31 - 1025):
        for cols in (32, 28672, 200_000, 400_000, 3_000_000):
            for kind in (blas.KIND_I8, blas.KIND_I16, blas.KIND_Q16):
                for experts in (0, 5):
                    assert 1 <= blas.w4_shape(kind, m, 4096, cols, 128, experts)["tries"] <= 6, (m, cols, kind, experts)


def test_addresses_of_operands():
    """Each kind of operand is recognised for what it is: an array is not first asked for a tensor's methods."""
    class Array(np.ndarray):
        def __getattr__(self, name):
            raise AssertionError(f"looked for {name}")

    a = np.arange(12, dtype=I32).reshape(3, 4)
    assert blas.addr(a.view(Array)) == blas.addr(a) == a.ctypes.data
    assert blas.addr(7) == 7 and blas.addr(np.int64(9)) == 9 and blas.addr(True) == 1
    with pytest.raises(ValueError):
        blas.addr(a.T)
    with pytest.raises(TypeError):
        blas.addr("a")
    torch = pytest.importorskip("torch")
    t = torch.zeros(3, 4)
    assert blas.addr(t) == t.data_ptr()
    with pytest.raises(ValueError):
        blas.addr(t.t())


OLDER_LIBRARY = """
#include <stdint.h>
typedef int64_t i;
#define SIX(n, v) i n(i a, i b, i c, i d, i e, i f) { (void)a, (void)b, (void)c, (void)d, (void)e, (void)f; return v; }
#define FIVE(n, v) i n(i a, i b, i c, i d, i e) { (void)a, (void)b, (void)c, (void)d, (void)e; return v; }
#define THREE(n, v) i n(i a, i b, i c) { (void)a, (void)b, (void)c; return v; }
SIX(__mind_blas_matmul_mm_i8_v, 1) SIX(__mind_blas_matmul_mm_i8_mt_v, 2) SIX(__mind_blas_matmul_mm_q16_v, 3)
SIX(__mind_blas_matmul_mm_q16_mt_v, 4) SIX(__mind_b200_matmul_mm_i16, 5)
FIVE(__mind_blas_gemv_q16_mt, 6) FIVE(__mind_blas_matmul_rmajor_q16_v, 7) FIVE(__mind_blas_matmul_rmajor_i16_v, 8)
THREE(__mind_blas_dot_q16_v, 9) THREE(__mind_blas_dot_l1_q16_v, 10) THREE(__mind_blas_dot_i16_v, 11)
const char *mind_b200_last_error(void) { return "the older library's own"; }
"""
OLDER_CHILD = r"""
import ctypes as C, sys
L = C.CDLL(sys.argv[1])
i64 = C.c_int64
def call(name, n):
    f = getattr(L, name); f.argtypes, f.restype = [i64] * n, i64
    return f(*[0] * n)
err = L.mind_b200_native_last_error; err.restype = C.c_char_p
for want, (name, n) in enumerate([("__mind_blas_matmul_mm_i8_v", 6), ("__mind_blas_matmul_mm_i8_mt_v", 6), ("__mind_blas_matmul_mm_q16_v", 6),
        ("__mind_blas_matmul_mm_q16_mt_v", 6), ("__mind_b200_matmul_mm_i16", 6), ("__mind_blas_gemv_q16_mt", 5),
        ("__mind_blas_matmul_rmajor_q16_v", 5), ("__mind_blas_matmul_rmajor_i16_v", 5), ("__mind_blas_dot_q16_v", 3),
        ("__mind_blas_dot_l1_q16_v", 3), ("__mind_blas_dot_i16_v", 3)], 1):
    assert call(name, n) == want, (name, err())
assert err() == b"the older library's own"
for n, names in {9: ["gemv_w4_i8", "gemv_w4_i16", "gemv_w4_q16"], 7: ["expert_plan"], 12: ["matmul_grouped_i8", "matmul_grouped_i8_bt"],
                 13: ["gemv_w4_grouped_i8", "gemv_w4_grouped_i16", "gemv_w4_grouped_q16"]}.items():
    for name in names:
        assert call("__mind_b200_" + name, n) == -3, name
        assert b"__mind_b200_" + name.encode() in err(), (name, err())
assert call("__mind_blas_matmul_mm_i8_v", 6) == 1 and err() == b"the older library's own"
print("ok")
"""


def test_native_sources_file_with_an_older_library(tmp_path):
    """A library that lacks the products of quantised language models serves everything else as before."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    shim, old = str(tmp_path / "libshim.so"), str(tmp_path / "libmind_b200.so")
    (tmp_path / "old.c").write_text(OLDER_LIBRARY)
    for out, src, libs in ((shim, os.path.join(root, "integration", "mind_b200_native.c"), ["-ldl", "-lpthread"]),
                           (old, str(tmp_path / "old.c"), [])):
        subprocess.run(["gcc", "-O2", "-Wall", "-Wextra", "-Werror", "-fPIC", "-shared", "-o", out, src, *libs], check=True)
    r = subprocess.run([sys.executable, "-c", OLDER_CHILD, shim], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, MIND_B200_LIB=old))
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr
