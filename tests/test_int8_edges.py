"""The int8 path where its calls go wrong most easily: views, broadcast dimensions, sizes at the ends of the range.

Bounds are those of test_int8_path.py: a product is an exact integer, three float32 roundings and the output's own; a normalised value
is good to REL = 2^-18."""
import contextlib
import ctypes
import itertools
import os
import random
import subprocess
import sys
import threading

import pytest
import torch

import locomp_b200 as L
from locomp_b200 import _lib, int8_ops
from test_int8_path import HALF_STEP, KINDS, NAMES, REL, check_product, check_tokens, gen, plan, product_case, rms, status_ok

tensor_module = sys.modules["locomp_b200.tensor"]        # (the package's `tensor` is a function)


# ------------------------------------------------------------------------------------------ views
def rows_apart(t):
    """By listing where every row starts: the distance between rows, where there is one that keeps them apart."""
    n = t.shape[-1]
    if n != 1 and t.stride(-1) != 1:
        return None
    starts = [sum(i * s for i, s in zip(at, t.stride())) for at in itertools.product(*map(range, t.shape[:-1]))]
    if len(starts) == 1:
        return n
    ld = starts[1] - starts[0]
    return ld if ld >= n and starts == [i * ld for i in range(len(starts))] else None


def test_row_stride_is_that_of_every_row():
    views = 0
    for shape in ((8,), (3, 8), (3, 4, 8), (2, 3, 2, 4), (3, 1, 8), (1, 3, 8), (3, 4, 1), (1, 1, 8)):
        steps = [(0, 1, 4, 8, 12, 16, 24, 32, 48, 96)] * (len(shape) - 1) + [(1, 2)]
        for strides in itertools.product(*steps):
            t = torch.empty(4096, dtype=torch.int8).as_strided(shape, strides)
            got, want = _lib.calls.row_stride(t), rows_apart(t)
            if all(s == 1 for s in shape[:-1]):           # a single row: any distance serves
                want = None if want is None else got
            assert got == want, (shape, strides, got, want)
            views += got is not None
    assert views > 50
    base = torch.zeros(3, 8)
    assert _lib.calls.row_stride(base[:, None].expand(3, 4, 8)) is None
    assert _lib.calls.row_stride(base[None].expand(4, 3, 8)) is None
    assert _lib.calls.row_stride(base[:, None, None].expand(3, 2, 2, 8)) is None
    assert _lib.calls.row_stride(base[:, :5]) == 8 and _lib.calls.row_stride(base[:, None]) == 8
    assert _lib.calls.row_stride(base.t()) is None and _lib.calls.row_stride(torch.zeros(())) is None


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_broadcast_rows_are_refused(kind):
    """Twelve rows of a storage that is cut out of a larger one, so that no stride leads out of it."""
    whole = torch.randn(64, 64, device="cuda", generator=gen(1)).to(kind)
    base = whole[:3, :]
    good = whole[:12].view(3, 4, 64)
    for x in (base[:, None].expand(3, 4, 64), base[None].expand(4, 3, 64), base[:1, None].expand(1, 4, 64)):
        with pytest.raises(ValueError, match="contiguous"):
            L.quantize_tokens(x)
        for gate, up in ((x, x), (good.reshape(x.shape) if x.numel() == good.numel() else x, x)):
            with pytest.raises(ValueError, match="contiguous"):
                L.silu_mul_tokens(gate, up)
    q = torch.full((64, 64), 5, dtype=torch.int8, device="cuda")
    s = torch.zeros(3, 4, device="cuda")
    w = torch.ones(64, device="cuda", dtype=kind)
    for out_q in (q[:3, None].expand(3, 4, 64), q[None, :4].expand(3, 4, 64)):
        t = L.QuantizedTokens(out_q, s)
        with pytest.raises(ValueError, match="contiguous"):
            L.quantize_tokens(good, out=t)
        with pytest.raises(ValueError, match="contiguous"):
            L.silu_mul_tokens(good, good, out=t)
        with pytest.raises(ValueError, match="contiguous"):
            L.residual_norms(good.clone(), good, w, quantized=True, out=t)
    assert bool((q == 5).all()) and bool((s == 0).all())
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_views_of_three_dimensions(kind):
    """Rows equally far apart over two dimensions are read and written where they are."""
    whole = torch.randn(3, 4, 80, device="cuda", generator=gen(2)).to(kind)
    x = whole[..., 8:72]
    t, want = L.quantize_tokens(x), L.quantize_tokens(x.contiguous())
    assert t.q.shape == (3, 4, 64) and torch.equal(t.q, want.q) and torch.equal(t.scales, want.scales)
    q = torch.full((3, 4, 96), 7, dtype=torch.int8, device="cuda")
    out = L.QuantizedTokens(q[..., :64], torch.empty(3, 4, device="cuda"))
    assert L.quantize_tokens(x, out=out) is out and torch.equal(out.q, want.q) and bool((q[..., 64:] == 7).all())
    s = L.silu_mul_tokens(x, x)
    assert torch.equal(s.q, L.silu_mul_tokens(x.contiguous(), x.contiguous()).q)
    with pytest.raises(ValueError, match="contiguous"):
        L.quantize_tokens(whole[:, :3, :64])          # four rows a block in storage, three of them taken: not equally far apart


# ------------------------------------------------------------------------------------------ kernels that share an SM
def test_no_successor_before_the_tensor_memory_is_taken():
    """A CTA that waits for columns of tensor memory must not have let the next kernel onto its SM: order of the source, since running
    it the other way round may hang a GPU."""
    for name in ("gemm_tc.cuh", "int8_gemm.cuh"):
        text = open(os.path.join(os.path.dirname(_lib.__file__), "csrc", name)).read()
        kernel = text[text.index("extern __shared__"):]
        kernel = kernel[:kernel.index("\n}\n")]
        places = [kernel.index(s) for s in ("tmem_alloc<CG>(tmem_slot", "__syncthreads();", "cluster_barrier();", "griddep_launch_dependents();")]
        assert places == sorted(places), name
        assert kernel.count("griddep_launch_dependents") == 1 and kernel.count("tmem_alloc<") == 1


def test_clusters_that_fit_on_an_sm_fit_into_its_tensor_memory():
    """Two clusters that meet on two SMs in opposite order, and do not fit there together, would wait for each other."""
    seen = {}
    r = random.Random(5)
    problems = [(692, 7513, 114), (412, 6844, 53), (38, 2663, 2811), (2049, 3000, 256), (512, 14336, 128)]
    problems += [(int(2 ** r.uniform(3, 11)), int(2 ** r.uniform(5, 13)), int(2 ** r.uniform(5, 12))) for _ in range(3000)]
    for m, n, k in problems:
        p = plan(m, n, k)
        if p["cg"] * p["split"] == 1:
            continue
        columns = 32
        while columns < p["bm"] + (p["bm"] + 31) // 32 * 32:          # two accumulators, the second read 32 columns at a time
            columns *= 2
        seen[columns] = min(seen.get(columns, 1 << 30), p["smem"] + 1024)      # 1 KB of a CTA is the system's
    assert 512 in seen and len(seen) > 2
    most = 228 * 1024
    for counts in itertools.product(*(range(most // s + 1) for s in seen.values())):
        if sum(c * s for c, s in zip(counts, seen.values())) <= most:
            assert sum(c * k for c, k in zip(counts, seen)) <= 512, (seen, counts)


@pytest.mark.gpu
def test_small_and_large_products_in_a_chain_and_on_two_streams():
    """Short rings, which leave room on an SM, one after the other and side by side."""
    sizes = [(16, 16384, 128), (1000, 3000, 128), (692, 7513, 114), (16, 16384, 128), (2048, 512, 144), (40, 2663, 2816)]
    cases = [product_case(*s) for s in sizes]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(60):
        outs.append((i % 6, L.int8_matmul(*cases[i % 6][:4], out_dtype="f32")))
    for i in range(60):
        outs.append((i // 2 % 6, L.int8_matmul(*cases[i // 2 % 6][:4], out_dtype="f32", stream=streams[i % 2])))
    torch.cuda.synchronize()
    first = {}
    for i, y in outs:
        if i not in first:
            check_product(y, cases[i][4], torch.float32)
        assert torch.equal(first.setdefault(i, y), y)
    status_ok()


# ------------------------------------------------------------------------------------------ sizes
def test_sizes_near_the_end_of_int_are_refused():
    """Within a tile of 2^31 the kernels' channel and token numbers would pass the end of int."""
    lib, f, p = _lib.lib(), (ctypes.c_int * 9)(), ctypes.c_void_p(4096)
    for m, n in ((1, 2000000000), (2000000000, 1)):
        assert lib.lcq_int8_matmul_workspace_bytes(m, n, 16, 1, 1) != (1 << 64) - 1
    for m, n in ((1, 2000000001), (1, 2 ** 31 - 1), (2 ** 31 - 1, 1), (2 ** 31 - 1, 2 ** 31 - 1)):
        assert lib.lcq_int8_matmul_workspace_bytes(m, n, 16, 1, 1) == (1 << 64) - 1
        assert lib.lcq_int8_matmul_plan_check(m, n, 16, 148, 1, f) == _lib.ERR_UNSUPPORTED
        assert lib.lcq_int8_matmul(p, 16, p, p, 16, p, p, m, n, 16, 0, 0, None, 0, None) == _lib.ERR_UNSUPPORTED


def test_sizes_that_an_int_does_not_hold_are_refused():
    """ctypes cuts an int to 32 bits: 2^32 + 8 values a row would run as 8, the others left as they were."""
    lib, p, big = _lib.lib(), ctypes.c_void_p(4096), 2 ** 32
    calls = [lambda: lib.lcq_int8_matmul(p, 16, p, p, 16, p, p, big, 0, 16, 0, 0, None, 0, None),
             lambda: lib.lcq_int8_matmul_workspace_bytes(0, big + 8, 16, 1, 1),
             lambda: lib.lcq_quantize_tokens(p, 8, None, p, 8, p, 0, big + 8, 1e-5, 0, None),
             lambda: lib.lcq_silu_mul_tokens(p, 8, p, 8, p, 8, p, 0, -big, 0, None),
             lambda: lib.lcq_residual_norms(p, p, None, None, 0, 1.0, None, p, None, 8, None, 0, big + 8, 1e-5, 0, None),
             lambda: lib.lcq_rms_norm(p, p, p, 0, 2 ** 31, 1e-5, 0, None)]
    for call in calls:
        with pytest.raises(ctypes.ArgumentError, match="does not fit"):
            call()
    assert lib.lcq_residual_norms(None, None, None, None, 0, 1.0, None, None, None, 0, None, big, 0, 1e-5, 0, None) == 0      # rows are 64 bits


def test_a_plan_without_the_memory_to_check_it_is_refused():
    """An exception may not leave a C entry: 62500 x 7813 pieces, in a process of little memory."""
    code = ("import ctypes, resource, sys\n"
            "lib = ctypes.CDLL(sys.argv[1])\n"
            "here = int(open('/proc/self/statm').read().split()[0]) * resource.getpagesize()\n"
            "resource.setrlimit(resource.RLIMIT_AS, (here + (1 << 29), resource.getrlimit(resource.RLIMIT_AS)[1]))\n"
            "sys.exit(10 + lib.lcq_int8_matmul_plan_check(1000000, 1000000, 64, 148, 1, None))\n")
    assert subprocess.run([sys.executable, "-c", code, _lib.LIB_PATH], timeout=120).returncode == 10 + _lib.ERR_UNSUPPORTED


@pytest.mark.gpu
def test_rows_that_an_int_does_not_hold_are_refused():
    n = 2 ** 32 + 8
    x = torch.zeros(1, n, dtype=torch.float16, device="cuda")
    for call in (lambda: L.quantize_tokens(x), lambda: L.silu_mul_tokens(x, x), lambda: L.residual_norms(x, x)):
        with pytest.raises(ctypes.ArgumentError, match="does not fit"):
            call()
    q = x.view(torch.int8)[:, :n]
    one = torch.ones(1, device="cuda")
    with pytest.raises(ctypes.ArgumentError, match="does not fit"):
        L.int8_matmul(q, one, q, one)


def test_weights_are_copied_48_mib_at_a_time_at_most():
    """Also where a piece's rows, rounded up to tiles, would be more."""
    lib = _lib.lib()
    for k in (17, 577, 4099, 14337, 60001, 131071):
        row = (k + 15) // 16 * 16
        for n in (3000, 385, 1000, 5003, 20000, 300000):
            counters = lib.lcq_int8_matmul_workspace_bytes(16, 1, 1, 1, 0) - 1024
            copied = lib.lcq_int8_matmul_workspace_bytes(16, n, k, 1, 0) - counters
            assert copied <= 48 << 20 and copied >= min(n * row, 24 << 20), (n, k, copied)
            p = plan(16, n, k, aligned=0)
            assert p["piece"] == n or p["piece"] % 256 == 0


def test_rows_of_no_values_have_no_scale():
    """They used to return with their scales left as they were."""
    lib, p, bad = _lib.lib(), ctypes.c_void_p(4096), _lib.ERR_BAD_ARG
    assert lib.lcq_quantize_tokens(p, 0, None, p, 0, p, 5, 0, 1e-5, 0, None) == bad
    assert lib.lcq_silu_mul_tokens(p, 0, p, 0, p, 0, p, 5, 0, 0, None) == bad
    assert lib.lcq_residual_norms(p, p, None, None, 0, 1.0, p, p, p, 0, p, 5, 0, 1e-5, 0, None) == bad
    assert lib.lcq_residual_norms(p, p, None, None, 0, 1.0, p, p, p, 0, None, 5, 0, 1e-5, 0, None) == 0
    for rows in (0, 5):
        assert lib.lcq_quantize_tokens(p, 8, None, p, 8, p, 0, rows, 1e-5, 0, None) == 0


@pytest.mark.gpu
def test_calls_on_nothing():
    for kind in KINDS:
        for shape in ((5, 0), (2, 3, 0), (0,)):
            x = torch.empty(shape, device="cuda", dtype=kind)
            for call in (lambda: L.quantize_tokens(x), lambda: L.silu_mul_tokens(x, x), lambda: L.quantize_tokens(x, x.reshape(-1)[:0]),
                         lambda: L.residual_norms(x, x, torch.empty(0, device="cuda", dtype=kind), quantized=True)):
                with pytest.raises(ValueError, match="no scale"):
                    call()
            assert L.residual_norms(x, x) is x
        none = torch.empty(0, 64, device="cuda", dtype=kind)
        w = torch.ones(64, device="cuda", dtype=kind)
        for t in (L.quantize_tokens(none, w), L.silu_mul_tokens(none, none), L.residual_norms(none, none, w, quantized=True)):
            assert t.q.shape == (0, 64) and t.scales.shape == (0,)
        assert L.residual_norms(none, none, w).shape == (0, 64)
        one = torch.ones(3, device="cuda")
        with pytest.raises(ValueError, match="K=0"):
            L.int8_matmul(torch.empty(3, 0, dtype=torch.int8, device="cuda"), one, torch.empty(3, 0, dtype=torch.int8, device="cuda"), one)


# ------------------------------------------------------------------------------------------ outputs and layers
def test_tokens_go_into_tokens():
    x = torch.zeros(4, 64)
    for call in (lambda out: L.quantize_tokens(x, out=out), lambda out: L.silu_mul_tokens(x, x, out=out)):
        for out in (torch.zeros(4, 64, dtype=torch.int8), (x, x), 3):
            with pytest.raises(TypeError, match="QuantizedTokens"):
                call(out)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,n,k", [((2, 3), 40, 100), ((1, 1), 40, 64), ((4, 1, 5), 300, 512), ((2, 150), 256, 333), ((8, 1), 64, 96)])
def test_batches_of_sequences(shape, n, k):
    """Tokens of more dimensions go through the product and the layer as their rows do."""
    g = gen(n, k)
    q = L.quantize(torch.randn(n, k, device="cuda", generator=g), k, bits=8)
    layer, w = q.int8_linear(), 1 + 0.1 * torch.randn(k, device="cuda", generator=g)
    x = torch.randn(*shape, k, device="cuda", generator=g)
    rows = x.numel() // k
    t = L.quantize_tokens(x)
    y = L.int8_matmul(t.q, t.scales, q.w, q.scales, out_dtype="f32")
    flat = L.quantize_tokens(x.view(rows, k))
    want = L.int8_matmul(flat.q, flat.scales, q.w, q.scales, out_dtype="f32")
    assert y.shape == shape + (n,) and torch.equal(y.view(rows, n), want)
    check_product(y.view(rows, n), flat.q.double() @ q.w.double().t() * flat.scales.double()[:, None] * q.scales.double().view(-1), torch.float32)
    assert torch.equal(layer(x), y) and torch.equal(layer(t, out_dtype="f32"), y)
    assert torch.equal(layer(x, w).view(rows, n), layer(x.view(rows, k), w))
    D = L.DeviceTensor                                       # the general path
    assert torch.equal(L.int8_matmul(D(t.q.contiguous()), t.scales, q.w, q.scales, out_dtype="f32"), y)
    out = torch.empty(shape + (n,), device="cuda")
    assert layer(x, out=out) is out and torch.equal(out, y)
    out = torch.empty(rows, n, device="cuda")
    assert L.int8_matmul(t.q, t.scales, q.w, q.scales, out=out) is out and torch.equal(out, want)
    wide = torch.randint(-128, 128, shape + (k + 16,), dtype=torch.int8, device="cuda", generator=g)[..., 5:5 + k]
    assert torch.equal(L.int8_matmul(wide, t.scales, q.w, q.scales, out_dtype="f32"),
                       L.int8_matmul(wide.contiguous(), t.scales, q.w, q.scales, out_dtype="f32"))
    for scales in (t.scales.reshape(-1), t.scales[None]):
        with pytest.raises(ValueError, match="must be \\[K\\]"):
            L.int8_matmul(t.q, scales, q.w, q.scales)
    with pytest.raises(ValueError, match="contiguous"):
        L.int8_matmul(t.q[:, :1].expand(t.q.shape) if shape[1] > 1 else t.q[:1].expand((3,) + t.q.shape[1:]),
                      t.scales if shape[1] > 1 else torch.ones((3,) + t.scales.shape[1:], device="cuda"), q.w, q.scales)
    empty = L.quantize_tokens(x[:0])
    assert layer(empty).shape == (0,) + shape[1:] + (n,)
    status_ok()


def test_a_stream_of_another_device_is_refused(monkeypatch):
    """Its context would make its device the current one, and the kernel would run there on this device's addresses."""
    class Stream:
        device, cuda_stream = torch.device("cuda", 1), 4096
    entered = []
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext(entered.append(s)))
    with pytest.raises(ValueError, match="stream on cuda:1"):
        with int8_ops._on(0, Stream()):
            pass
    assert not entered
    with int8_ops._on(1, Stream()):
        assert len(entered) == 1


@pytest.mark.gpu
def test_a_layer_of_weights_whose_rows_lie_on_one_another():
    """A broadcast weight is copied, as every other whose rows the product cannot read in place; it was kept, and every call refused it."""
    g = gen(3)
    row = torch.randint(-127, 128, (1, 64), dtype=torch.int8, device="cuda", generator=g)
    scales, x = torch.rand(24, device="cuda", generator=g), torch.randn(5, 64, device="cuda", generator=g)
    for w in (row.expand(24, 64), torch.randint(-127, 128, (48 + 23 * 16,), dtype=torch.int8, device="cuda", generator=g).as_strided((24, 48), (16, 1)),
              torch.randint(-127, 128, (64, 24), dtype=torch.int8, device="cuda", generator=g).t()):
        k = w.shape[1]
        assert torch.equal(L.Int8Linear(w, scales)(x[:, :k].contiguous()), L.Int8Linear(w.contiguous(), scales)(x[:, :k].contiguous()))
    status_ok()


# ------------------------------------------------------------------------------------------ float32 between operators
MIXED = [(1, 1), (1, 576), (5, 100), (9, 512), (2, 513), (7, 1537), (4, 4096), (33, 264), (1, 8192), (3, 8200), (2, 16384), (3, 16392), (2, 20001), (1, 50000),
         (600, 64), (1200, 1537), (400, 2048)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS[1:])
@pytest.mark.parametrize("rows,n", MIXED)
def test_residual_of_a_float32_delta(rows, n, kind):
    """hidden of 16 bits, delta as a product leaves it in float32: rounded once, as the sum is stored.  Bounds as in test_rows_against_64_bits."""
    g = gen(rows, n)

    def draw(r, scale=1.0, plus=0.0, as_kind=kind):
        return (torch.randn(r, n, device="cuda", generator=g) * scale + plus).to(as_kind)
    x, delta, w, post = draw(rows), draw(rows, 3.0, 0.0, torch.float32), draw(1, 0.1, 1.0)[0], draw(1, 0.1, 1.0)[0]
    for has_post, gate_rows, scale in ((True, 1, 0.5), (False, rows, -1.5), (True, 0, 1.0), (False, 0, 1.0)):
        gate = draw(gate_rows, 0.5) if gate_rows else None
        kw = dict(gate=gate, post_weight=post if has_post else None, scale=scale)
        y = rms(delta.double(), post) if has_post else delta.double()
        if gate_rows:
            y = y * gate.double()
        y = scale * y
        ref = x.double() + y
        hidden = torch.empty_like(x)
        out = L.residual_norms(x, delta, w, hidden_out=hidden, **kw)
        assert out.dtype == kind
        slack = REL * y.abs() + 2.0 ** -24 * ref.abs()
        assert bool(((hidden.double() - ref).abs() <= HALF_STEP[kind] * ref.abs() + (1 + HALF_STEP[kind]) * slack + 2.0 ** -25).all())
        normed = rms(hidden.double(), w)
        assert bool(((out.double() - normed).abs() <= (HALF_STEP[kind] + 1.01 * REL) * normed.abs() + 2.0 ** -25).all())
        again = x.clone()
        tokens = L.residual_norms(again, delta, w, quantized=True, **kw)
        assert torch.equal(again, hidden)
        check_tokens(tokens, normed)
        once = x.clone()
        assert L.residual_norms(once, delta, **kw) is once and torch.equal(once, hidden)
        if has_post and gate_rows:                            # the general path, and rows off 16 bytes
            once = x.clone()
            assert torch.equal(L.residual_norms(L.DeviceTensor(once), delta, w, **kw), out) and torch.equal(once, hidden)
            off = torch.empty(rows * n + 1, device="cuda")[1:].view(rows, n).copy_(delta)
            once = x.clone()
            moved = L.residual_norms(once, off, w, **kw)
            assert bool(((once.double() - ref).abs() <= HALF_STEP[kind] * ref.abs() + (1 + HALF_STEP[kind]) * slack + 2.0 ** -25).all())
            normed = rms(once.double(), w)
            assert bool(((moved.double() - normed).abs() <= (HALF_STEP[kind] + 1.01 * REL) * normed.abs() + 2.0 ** -25).all())
    status_ok()


@pytest.mark.gpu
def test_residual_refuses_other_types_of_delta():
    f = {k: torch.randn(4, 64, device="cuda").to(k) for k in KINDS}
    for hidden in KINDS:
        for delta in KINDS:
            if delta in (hidden, torch.float32):
                assert L.residual_norms(f[hidden].clone(), f[delta], f[hidden][0]).dtype == hidden
            else:
                with pytest.raises(TypeError, match="delta must be"):
                    L.residual_norms(f[hidden].clone(), f[delta], f[hidden][0])
            if delta != hidden:                               # nothing else may differ
                for kw in (dict(weight=f[delta][0]), dict(post_weight=f[delta][0]), dict(gate=f[delta][0]), dict(hidden_out=f[delta].clone()),
                           dict(weight=f[hidden][0], out=f[delta].clone())):
                    with pytest.raises(TypeError, match="one dtype"):
                        L.residual_norms(f[hidden].clone(), f[hidden], **kw)
    with pytest.raises(TypeError, match="delta must be"):
        L.residual_norms(f[torch.float16].clone(), torch.zeros(4, 64, dtype=torch.int8, device="cuda"))


def test_residual_entry_checks_the_type_of_delta():
    lib, p = _lib.lib(), ctypes.c_void_p(4096)
    for dtype in range(3):
        for delta in range(-1, 5):
            rc = lib.lcq_residual_norms_delta(p, p, delta, None, None, 0, 1.0, p, p, p, 8, None, 0, 8, 1e-5, dtype, None)
            assert rc == (0 if delta in (dtype, 0) else _lib.ERR_BAD_ARG)
    assert lib.lcq_residual_norms_delta(p, p, 0, None, p, 4, 1.0, p, p, p, 8, None, 6, 8, 1e-5, 1, None) == _lib.ERR_BAD_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS[1:])
def test_decode_stack_rounds_where_something_is_stored(kind):
    """From tokens to tokens and to the stream against 64 bits, across the product and what follows it: nothing is rounded to 16 bits between."""
    inter = 1536
    st = L.DecodeStack(layers=1, hidden=576, inter=inter, vocab=1000, fused=True, glue=True, int8=True, dtype=kind, post_norms=True, residual_scale=0.5, seed=2)
    assert [out.dtype for _, _, out in st.calls] == [torch.float32] * 4 + [kind]
    st.token.fill_(7)
    ops, norms, calls = iter(st.ops), iter(st.norms), iter(st.calls)

    def product():
        lin, tokens, _ = next(calls)
        next(ops)()
        return tokens.q.double() @ lin.w.double().t() * tokens.scales.double()[:, None] * lin.scales.double()

    def block_end(delta):
        before = st.hidden.double()
        next(ops)()
        y = 0.5 * rms(delta, next(norms))
        ref = before + y
        # a product in float32 is off by 3 * 2^-24, its norm by REL and less than that again
        assert bool(((st.hidden.double() - ref).abs() <= HALF_STEP[kind] * ref.abs() + (1 + HALF_STEP[kind]) * (2 * REL * y.abs() + 2.0 ** -24 * ref.abs()) + 2.0 ** -25).all())
        check_tokens(st.normed, rms(st.hidden.double(), next(norms)))
    next(ops)()
    next(ops)()
    next(norms)
    product()
    block_end(product())
    gu = product()
    next(ops)()
    a, b = gu[:, :inter], gu[:, inter:]
    check_tokens(st.mlp, a * torch.sigmoid(a) * b)
    block_end(product())
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS[1:])
def test_half_way_quotients_of_normed_tokens(kind):
    """Of 16-bit rows x weight is exact, and quotients v / (amax / 127) that are half-integers are common.  No float32 scale makes all of them ties to even
    (a float32 division has 15 % of those of amax / 2 wrong, over all 8-bit amax), but a reciprocal without the quotient's rounding had half."""
    g = gen(11)
    x = torch.randn(20000, 512, device="cuda", generator=g).to(torch.bfloat16).to(kind)          # 8 bits of mantissa in either type
    w = torch.tensor([0.5, 1.0, 2.0], device="cuda", dtype=kind)[torch.randint(0, 3, (512,), device="cuda", generator=g)]
    v = x.double() * w.double()
    amax = v.abs().amax(-1, keepdim=True)
    half = (254 * v / amax).round()
    ties = (half * amax == 254 * v) & (half.remainder(2) == 1)
    even = (127 * v[ties] / amax.expand_as(v)[ties]).round()
    assert int(ties.sum()) > 500
    for t in (L.quantize_tokens(x, w), L.residual_norms(torch.zeros_like(x), x, w, quantized=True)):
        check_tokens(t, rms(x.double(), w))
        assert int((t.q[ties].double() != even).sum()) <= 0.25 * int(ties.sum())
    status_ok()


# ------------------------------------------------------------------------------------------ long rows
@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_millions(kind):
    """One bound for rows of any length: equal values, whose rounding errors all have one sign in a running sum."""
    for n, value in ((1 << 22, 1.1), (1 << 24, 0.7), ((1 << 24) + 3, 1.7)):
        x = torch.full((1, n), value, device="cuda").to(kind)
        ramp = (1 + (torch.arange(n, device="cuda") % 5) * 0.25).to(kind)
        want = rms(x.double(), ramp)
        check_tokens(L.quantize_tokens(x, ramp), want)
        hidden = torch.zeros_like(x)
        out = L.residual_norms(hidden, x, ramp, post_weight=torch.ones_like(ramp))
        assert bool(((hidden.double() - rms(x.double(), torch.ones_like(ramp))).abs() <= HALF_STEP[kind] + (1 + HALF_STEP[kind]) * REL).all())
        normed = rms(hidden.double(), ramp)
        assert bool(((out.double() - normed).abs() <= (HALF_STEP[kind] + 1.01 * REL) * normed).all())
        del want, normed
    status_ok()


# longer than a block's registers hold in any type
LONG = [(2, 32769), (1, 40001), (3, 50003), (2, 65537 + 6)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n", LONG)
@pytest.mark.parametrize("place", [0, 1, 5])
def test_long_rows_off_16_bytes(rows, n, kind, place):
    """Rows that are read again for each pass over them, written from the first value on 16 bytes on, at other places in every operand.  Bounds as in
    test_rows_against_64_bits."""
    g = gen(rows, n, place)

    def draw(r, scale=1.0, plus=0.0, at=0):
        flat = torch.empty(r * n + 8, device="cuda", dtype=kind)
        return flat[at:at + r * n].view(r, n).copy_(torch.randn(r, n, device="cuda", generator=g) * scale + plus)
    x, delta = draw(rows, at=place), draw(rows, 3.0, at=(place + 3) % 8)
    w, post, gate = draw(1, 0.1, 1.0, at=(place + 1) % 8)[0], draw(1, 0.1, 1.0, at=place)[0], draw(rows, 0.5, at=(place + 2) % 8)
    t = L.quantize_tokens(x)
    whole = L.quantize(x.clone(), n, bits=8)
    assert torch.equal(t.q, whole.w) and torch.equal(t.scales, whole.scales.view(-1))
    check_tokens(L.quantize_tokens(x, w), rms(x.double(), w))
    a, b = x.double(), delta.double()
    check_tokens(L.silu_mul_tokens(x, delta), a * torch.sigmoid(a) * b)
    q = torch.full((rows, n + 32), 77, dtype=torch.int8, device="cuda")
    out = L.QuantizedTokens(q[:, 3:3 + n], torch.empty(rows, device="cuda"))
    L.silu_mul_tokens(x, delta, out=out)
    check_tokens(out, a * torch.sigmoid(a) * b)
    assert bool((q[:, :3] == 77).all()) and bool((q[:, 3 + n:] == 77).all())
    for has_post, gated, scale in ((True, True, 0.5), (False, True, -1.5), (True, False, 1.0), (False, False, 1.0)):
        kw = dict(post_weight=post if has_post else None, gate=gate if gated else None, scale=scale)
        y = rms(b, post) if has_post else b
        y = scale * (y * gate.double() if gated else y)
        ref = a + y
        buf = torch.full((rows * n + 16,), 9.0, device="cuda", dtype=kind)
        hidden = buf[7:7 + rows * n].view(rows, n)
        norm = torch.full((rows * n + 16,), 9.0, device="cuda", dtype=kind)
        written = norm[2:2 + rows * n].view(rows, n)
        assert L.residual_norms(x, delta, w, hidden_out=hidden, out=written, **kw) is written
        slack = REL * y.abs() + 2.0 ** -24 * ref.abs()
        assert bool(((hidden.double() - ref).abs() <= HALF_STEP[kind] * ref.abs() + (1 + HALF_STEP[kind]) * slack + 2.0 ** -25).all())
        normed = rms(hidden.double(), w)
        assert bool(((written.double() - normed).abs() <= (HALF_STEP[kind] + 1.01 * REL) * normed.abs() + 2.0 ** -25).all())
        for edge in (buf[:7], buf[7 + rows * n:], norm[:2], norm[2 + rows * n:]):
            assert bool((edge == 9).all())
        again = x.clone()
        check_tokens(L.residual_norms(again, delta, w, quantized=True, **kw), rms(again.double(), w))
        # (not the bits of `hidden`: octets are counted from where the written row lies on 16 bytes, so the squares of delta meet in another order and each
        # result has the bound above by itself)
        assert bool(((again.double() - ref).abs() <= HALF_STEP[kind] * ref.abs() + (1 + HALF_STEP[kind]) * slack + 2.0 ** -25).all())
        assert has_post or torch.equal(again, hidden)                    # no sum comes before hidden without the norm of delta
    status_ok()


# ------------------------------------------------------------------------------------------ one after the other
@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 8192, 2048), (1, 40000, 576), (4, 8192, 2048), (4, 8192, 2041), (16, 8192, 2048), (300, 8192, 2048), (300, 3000, 2041), (16, 9000, 2041)])
def test_product_of_operands_that_a_kernel_ahead_is_still_writing(m, n, k):
    """Weights, tokens and both scales come from kernels that let their successor start before they have written anything: each of the product's kernels (dp4a, warp MMAs,
    the ring, and the copy of rows off 16 bytes) has to wait for them.  Other values each time."""
    g = gen(m, n, k)
    weights = [torch.randn(n, k, device="cuda", generator=g) for _ in range(3)]
    tokens = [torch.randn(m, k, device="cuda", generator=g) for _ in range(2)]
    want = []
    for i in range(6):
        x, w = L.quantize_tokens(tokens[i % 2]), L.quantize_tokens(weights[i % 3])
        want.append(x.q.double() @ w.q.double().t() * x.scales.double()[:, None] * w.scales.double())
    w = L.QuantizedTokens(torch.zeros(n, k, dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda"))
    x = L.quantize_tokens(tokens[0])
    outs = torch.empty(24, m, n, device="cuda")

    def chain():
        for i in range(24):
            if i % 4 < 2:                                     # now the weights last, now the tokens
                L.quantize_tokens(tokens[i % 2], out=x)
                L.quantize_tokens(weights[i % 3], out=w)
            else:
                L.quantize_tokens(weights[i % 3], out=w)
                L.quantize_tokens(tokens[i % 2], out=x)
            L.int8_matmul(x.q, x.scales, w.q, w.scales, out=outs[i])
    torch.cuda.synchronize()
    chain()
    for i in range(24):
        check_product(outs[i], want[i % 6], torch.float32)
    direct = outs.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        chain()
    for _ in range(2):
        outs.zero_()
        graph.replay()
        assert torch.equal(outs, direct)
    status_ok()


@pytest.mark.gpu
def test_a_threads_first_call():
    """A thread that has made no CUDA call yet has no context, which the driver wants for a tensor map."""
    g = gen(12)
    w4 = torch.randint(0, 256, (2048, 512), dtype=torch.uint8, device="cuda", generator=g)
    s4 = (torch.rand(2048, 32, device="cuda", generator=g) * 0.02).half()
    calls = []
    for m in (1, 16, 300):
        a = torch.randn(m, 1024, device="cuda", generator=g).half()
        calls.append((lambda out, a=a: L.quantized_matmul(a, w4, s4, 32, out=out), L.quantized_matmul(a, w4, s4, 32)))
    for size in ((1, 512, 1024), (8, 512, 1024), (16, 512, 1024), (300, 512, 1024), (16, 512, 1001), (300, 512, 1001)):
        x, xs, w, ws, _ = product_case(*size)
        calls.append((lambda out, c=(x, xs, w, ws): L.int8_matmul(*c, out=out), L.int8_matmul(x, xs, w, ws)))
    x = torch.randn(4, 512, device="cuda", generator=g).half()
    norm = torch.ones(512, device="cuda").half()
    calls.append((lambda out: L.residual_norms(x, x, norm, hidden_out=torch.empty_like(x), out=out), L.residual_norms(x, x, norm, hidden_out=torch.empty_like(x))))
    torch.cuda.synchronize()
    for call, want in calls:
        out, failed = torch.zeros_like(want), []
        torch.cuda.synchronize()

        def work():
            try:
                call(out)
            except Exception as e:
                failed.append(e)
        t = threading.Thread(target=work)
        t.start()
        t.join()
        assert not failed, failed
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    status_ok()


@pytest.mark.gpu
def test_product_leaves_the_streams_scratch_to_the_graphs_that_hold_it():
    """A graph of int4 products holds the address of its stream's scratch.  The int8 product's copies used to make that buffer grow, which gave the old one to whoever
    allocated next."""
    g, side = gen(13), torch.cuda.Stream()
    w4 = torch.randint(0, 256, (20000, 2048), dtype=torch.uint8, device="cuda", generator=g)
    s4 = (torch.rand(20000, 128, device="cuda", generator=g) * 0.02).half()
    a = torch.randn(16, 4096, device="cuda", generator=g).half()
    want, out = L.quantized_matmul(a, w4, s4, 32), torch.empty(16, 20000, dtype=torch.float16, device="cuda")
    x, xs, w, ws, ref = product_case(16, 9000, 4101)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        L.quantized_matmul(a, w4, s4, 32, out=out)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            L.quantized_matmul(a, w4, s4, 32, out=out)
        before = {k: t.data_ptr() for k, t in tensor_module._workspaces.items()}
        for form in (x, L.DeviceTensor(x)):
            check_product(L.int8_matmul(form, xs, w, ws, out_dtype="f32"), ref, torch.float32)
            check_product(L.int8_matmul(form, xs, w, ws, out_dtype="f32", stream=side), ref, torch.float32)
        canaries = [torch.full((1 << 18,), 5, dtype=torch.int32, device="cuda") for _ in range(8)]
        out.zero_()
        for _ in range(3):
            graph.replay()
        side.synchronize()
    assert {k: t.data_ptr() for k, t in tensor_module._workspaces.items()} == before
    assert torch.equal(out, want) and all(bool((c == 5).all()) for c in canaries)
    status_ok()


@pytest.mark.gpu
def test_products_that_copy_share_a_stream_and_two_graphs():
    """Copies of two threads on one stream, and of two graphs that are replayed side by side: each has memory of its own."""
    cases = [product_case(m, n, k) for m, n, k in ((16, 9000, 2049), (40, 5000, 1001), (300, 3000, 577))]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    for x, xs, w, ws, _ in cases:
        outs.append(L.int8_matmul(x, xs, w, ws, out_dtype="f32"))
        graphs.append(torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(graphs[-1]):
            for _ in range(4):
                L.int8_matmul(x, xs, w, ws, out=outs[-1])
    for _ in range(10):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for y, case in zip(outs, cases):
        check_product(y, case[4], torch.float32)
    wrong = []

    def work(i):
        ys = [L.int8_matmul(*cases[(i + j) % 3][:4], out_dtype="f32") for j in range(30)]
        torch.cuda.current_stream().synchronize()
        wrong.extend((i, j) for j, y in enumerate(ys) if not torch.equal(y, outs[(i + j) % 3]))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 3])
def test_few_tokens_on_either_side_of_each_kernels_range(m):
    """One or two tokens go to dp4a, but for many rows of 1025 to 4095 bytes; three to warp MMAs up to 20 Mi weights.  Sizes next to each border."""
    for k, n in ((1024, 32768), (1025, 33000), (1040, 32264), (1040, 32263), (2048, 16384), (2048, 16383), (4080, 8224), (4095, 8300), (4096, 8192), (4096, 5120), (4096, 5121)):
        x, xs, w, ws, ref = product_case(m, n, k, torch.float16, pad=-k % 16)            # rows on 16 bytes
        check_product(L.int8_matmul(x, xs, w, ws, out_dtype="f32"), ref, torch.float32)
    status_ok()
