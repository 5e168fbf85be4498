"""The int8 path: tokens quantised a row at a time, products of int8 tokens and int8 weights, norms around a block.

Bounds.  A product is an exact integer sum S (|S| < 2^31), converted to float32 and multiplied by two float32 scales: three
roundings of 2^-24, then the output's own (2^-24, 2^-11, 2^-8 relative; float16 subnormals 2^-25 absolute).
Rows: float32 arithmetic on a sum of n squares.  A sum of n terms in float32 is off by at most (n / T + 10) 2^-24 relative with T
partial sums (no thread adds more than 32 squares here before the tree of ten steps); rsqrtf is good to 2 units of 2^-24; with
the products that makes less than 64 * 2^-24 = 2^-18 relative for a normalised value.  The residual is hidden + scale * y: its error
is that of y (two norms' worth at most) plus the storage rounding.
Tokens: q may differ from the 64-bit result by 1 where the quotient lies within 127 * 2^-18 of a half-integer, and nowhere else.
"""
import ctypes
import random
import threading

import pytest
import torch

import locomp_b200 as L
from locomp_b200 import _lib
from locomp_b200.int8_ops import int8_matmul_workspace_bytes

KINDS = [torch.float32, torch.float16, torch.bfloat16]
NAMES = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}
HALF_STEP = {k: torch.finfo(k).eps / 2 for k in KINDS}
REL = 2.0 ** -18


def gen(*seed):
    return torch.Generator(device="cuda").manual_seed(sum(31 ** i * int(s) for i, s in enumerate(seed)) % (1 << 31))


def status_ok():
    assert _lib.lib().lcq_check_device_status(None) == 0, _lib.lib().lcq_last_error()


# ------------------------------------------------------------------------------------------ the product's schedule (CPU)
def plan(m, n, k, sms=148, aligned=1):
    f = (ctypes.c_int * 9)()
    assert _lib.lib().lcq_int8_matmul_plan_check(m, n, k, sms, aligned, f) == 0, (m, n, k, sms, aligned, _lib.lib().lcq_last_error())
    return dict(zip(("ctas", "bm", "tiles", "in_pieces", "smem", "cg", "split", "depth", "piece"), f))


def test_plan_covers_every_stage_once():
    for m in (1, 2, 16, 17, 33, 64, 100, 256, 257, 512, 1000, 8192):
        for n in (1, 100, 128, 129, 2048, 5003, 28672):
            for k in (1, 64, 128, 129, 576, 4104, 14336):
                for sms in (148, 132, 7, 1):
                    for aligned in (0, 1):
                        plan(m, n, k, sms, aligned)
    r = random.Random(1)
    for _ in range(1500):
        plan(int(2 ** r.uniform(0, 13)), int(2 ** r.uniform(0, 15.5)), int(2 ** r.uniform(0, 17)) - 1 or 1, r.choice((148, 148, 132, 16)), r.choice((0, 1)))


def test_plan_refuses_what_the_product_refuses():
    lib, f = _lib.lib(), (ctypes.c_int * 9)()
    assert lib.lcq_int8_matmul_plan_check(1, 1, 131071, 148, 1, f) == 0
    assert lib.lcq_int8_matmul_plan_check(1, 1, 131072, 148, 1, f) == _lib.ERR_UNSUPPORTED
    assert lib.lcq_int8_matmul_plan_check(1, 1, 0, 148, 1, f) == _lib.ERR_BAD_ARG
    assert lib.lcq_int8_matmul_plan_check(2000000000, 2000000000, 64, 148, 1, f) == _lib.ERR_UNSUPPORTED
    assert lib.lcq_int8_matmul_workspace_bytes(1, 1, 131072, 1, 1) == (1 << 64) - 1 == lib.lcq_int8_matmul_workspace_bytes(-1, 1, 64, 1, 1)
    assert lib.lcq_int8_matmul_workspace_bytes(0, 1, 64, 1, 1) == 0
    with pytest.raises(ValueError):
        int8_matmul_workspace_bytes(1, 1, 1 << 20)


def test_c_entries_check_their_arguments():
    """Every refusal before the device is touched: pointers are never read."""
    lib, p, bad = _lib.lib(), ctypes.c_void_p(4096), _lib.ERR_BAD_ARG
    assert lib.lcq_int8_matmul(p, 64, p, p, 64, p, p, -1, 8, 64, 0, 0, None, 0, None) == bad
    assert lib.lcq_int8_matmul(p, 64, p, p, 64, p, p, 8, 8, 64, 3, 0, None, 0, None) == bad
    assert lib.lcq_int8_matmul(p, 64, p, p, 64, p, p, 8, 8, 64, 0, 7, None, 0, None) == bad
    assert lib.lcq_int8_matmul(None, 64, p, p, 64, p, p, 8, 8, 64, 0, 0, None, 0, None) == bad
    assert lib.lcq_int8_matmul(p, 63, p, p, 64, p, p, 8, 8, 64, 0, 0, None, 0, None) == bad
    assert lib.lcq_int8_matmul(p, 64, p, p, 63, p, p, 8, 8, 64, 0, 0, None, 0, None) == bad
    assert lib.lcq_int8_matmul(p, 64, p, p, 64, p, p, 0, 8, 64, 0, 0, None, 0, None) == 0
    assert lib.lcq_quantize_tokens(p, 8, None, p, 8, p, -1, 8, 1e-5, 0, None) == bad
    assert lib.lcq_quantize_tokens(p, 7, None, p, 8, p, 2, 8, 1e-5, 0, None) == bad
    assert lib.lcq_quantize_tokens(p, 8, None, p, 7, p, 2, 8, 1e-5, 0, None) == bad
    assert lib.lcq_quantize_tokens(p, 8, None, p, 8, None, 2, 8, 1e-5, 0, None) == bad
    assert lib.lcq_quantize_tokens(p, 8, None, p, 8, p, 2, 8, 1e-5, 9, None) == bad
    assert lib.lcq_quantize_tokens(p, 8, None, p, 8, p, 1, (1 << 30) + 1, 1e-5, 0, None) == _lib.ERR_UNSUPPORTED
    assert lib.lcq_quantize_tokens(None, 0, None, None, 0, None, 0, 8, 1e-5, 0, None) == 0
    assert lib.lcq_silu_mul_tokens(p, 8, p, 7, p, 8, p, 2, 8, 0, None) == bad
    assert lib.lcq_silu_mul_tokens(p, 8, None, 8, p, 8, p, 2, 8, 0, None) == bad
    args = [p, p, None, None, 0, 1.0, p, p, p, 8, None, 6, 8, 1e-5, 0, None]

    def norms(**kw):
        names = ["hidden", "delta", "post", "gate", "gate_rows", "scale", "weight", "hidden_out", "out", "ld_out", "scales", "rows", "n", "eps", "dtype", "stream"]
        return lib.lcq_residual_norms(*[kw.get(k, v) for k, v in zip(names, args)])
    assert norms(gate=p, gate_rows=4) == bad and norms(gate=p, gate_rows=0) == bad      # six rows
    assert norms(out=None) == bad and norms(hidden_out=None) == bad and norms(delta=None) == bad
    assert norms(weight=None, scales=p) == bad
    assert norms(ld_out=7) == bad and norms(n=-1) == bad and norms(dtype=5) == bad
    assert norms(rows=0, hidden=None) == 0


def test_what_is_not_a_cuda_tensor_is_refused_by_name():
    c, t, i = _lib.calls, torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.int8)
    assert c.quantize_tokens(t, None, 1e-5, None) is NotImplemented
    assert c.silu_mul_tokens(t, t, None) is NotImplemented
    assert c.residual_norms(t, t, None, 1e-5, None, None, 1.0, None, None, False) is NotImplemented
    assert c.int8_matmul(i, t, i, t, None, -1, None) is NotImplemented
    for call in (lambda: L.quantize_tokens(t), lambda: L.silu_mul_tokens(t, t), lambda: L.residual_norms(t, t), lambda: L.int8_matmul(i, t, i, t)):
        with pytest.raises(TypeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="CUDA"):
        L.Int8Linear(i, t[:, 0])


# ------------------------------------------------------------------------------------------ the product
def int8_rows(g, rows, k, pad=0, offset=0):
    wide = torch.randint(-128, 128, (rows, k + pad), dtype=torch.int8, device="cuda", generator=g)
    return wide[:, offset:offset + k]


def product_case(m, n, k, scale_kind=torch.float32, pad=0, offset=0):
    g = gen(m, n, k, pad, offset)
    x, w = int8_rows(g, m, k, pad, offset), int8_rows(g, n, k, pad, offset)
    xs = torch.rand(m, device="cuda", generator=g) * 0.02 + 0.01
    ws = (torch.rand(n, device="cuda", generator=g) * 0.01 + 0.001).to(scale_kind)
    return x, xs, w, ws, x.double() @ w.double().t() * xs.double()[:, None] * ws.double()


def check_product(y, ref, kind):
    bound = (3 * 2.0 ** -24 + HALF_STEP[kind]) * 1.001 * ref.abs() + (2.0 ** -25 if kind == torch.float16 else 0.0)
    over = ref.abs() > 65504 if kind == torch.float16 else torch.zeros_like(ref, dtype=torch.bool)
    assert bool((((y.double() - ref).abs() <= bound) | over).all())
    assert bool((y[over].float().abs() >= 65504).all())


PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 2048, 2048), (2, 130, 64), (3, 5, 16), (16, 28672, 1024), (17, 129, 144), (1, 49152, 576), (5, 4096, 14336),
            (31, 257, 1040), (32, 1000, 576), (33, 300, 512), (64, 5000, 4096), (100, 77, 2064), (128, 512, 4096), (255, 384, 272), (256, 2048, 4096),
            (257, 1001, 1024), (512, 9000, 768), (1000, 2048, 8192), (1025, 513, 640), (2049, 3000, 256), (4096, 128, 1024), (700, 20000, 512)]
UNALIGNED = [(1, 1, 7), (1, 300, 100), (5, 200, 333), (333, 1003, 1032), (64, 1000, 577), (1, 9000, 577), (200, 300, 17), (129, 130, 1), (16, 3000, 4104), (600, 700, 2049), (3, 50001, 1001), (40, 14000, 4099)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", PRODUCTS + UNALIGNED)
def test_product_against_64_bits(m, n, k):
    x, xs, w, ws, ref = product_case(m, n, k)
    for kind in KINDS:
        y = L.int8_matmul(x, xs, w, ws, out_dtype=NAMES[kind])
        assert y.shape == (m, n) and y.dtype == kind
        check_product(y, ref, kind)
        assert torch.equal(L.int8_matmul(x, xs, w, ws, out_dtype=NAMES[kind]), y)      # whoever adds the shares up
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("scale_kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pad,offset", [(0, 0), (16, 0), (16, 16), (16, 3), (12, 0), (5, 2)])
def test_product_rows_apart_and_types_of_scales(pad, offset, scale_kind):
    for m, n, k in ((1, 260, 512), (40, 300, 496), (300, 1000, 528)):
        x, xs, w, ws, ref = product_case(m, n, k, scale_kind, pad, offset)
        check_product(L.int8_matmul(x, xs, w, ws.view(n, 1), out_dtype="f32"), ref, torch.float32)
        check_product(L.int8_matmul(x[0], xs[:1], w, ws, out_dtype="f16"), ref[0], torch.float16)
    status_ok()


@pytest.mark.gpu
def test_product_is_exact_at_the_ends_of_int32():
    k = 131071
    for a, b in ((-128, -128), (127, -128), (127, 127)):
        x = torch.full((3, k), a, dtype=torch.int8, device="cuda")
        w = torch.full((130, k), b, dtype=torch.int8, device="cuda")
        one = torch.ones(130, device="cuda")
        y = L.int8_matmul(x, one[:3], w, one, out_dtype="f32")
        assert bool((y == torch.tensor(float(a * b * k), dtype=torch.float32)).all())
    with pytest.raises(_lib.LcqError, match="int32"):
        L.int8_matmul(torch.zeros(1, k + 1, dtype=torch.int8, device="cuda"), one[:1], torch.zeros(2, k + 1, dtype=torch.int8, device="cuda"), one[:2])
    status_ok()


@pytest.mark.gpu
def test_a_poisoned_token_stays_in_its_row():
    x, xs, w, ws, ref = product_case(20, 200, 256)
    xs[7], xs[9] = float("nan"), float("inf")
    y = L.int8_matmul(x, xs, w, ws, out_dtype="f32")
    keep = [i for i in range(20) if i not in (7, 9)]
    check_product(y[keep], ref[keep], torch.float32)
    assert bool(y[7].isnan().all()) and not bool(y[9].isfinite().any())


@pytest.mark.gpu
def test_product_writes_its_rows_and_nothing_else():
    for m, n, k in ((5, 300, 512), (300, 5000, 256), (70, 130, 333)):
        x, xs, w, ws, ref = product_case(m, n, k)
        buf = torch.full((m + 2, n), 3.0, device="cuda")
        out = buf[1:m + 1]
        assert L.int8_matmul(x, xs, w, ws, out=out) is out
        check_product(out, ref, torch.float32)
        assert bool((buf[0] == 3).all()) and bool((buf[-1] == 3).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(300, 257, 64), (77, 258, 640), (130, 131, 33), (64, 516, 32), (257, 391, 144), (1000, 255, 272), (33, 1029, 16), (150, 384, 96), (600, 3001, 128)])
def test_product_at_every_place_in_16_bytes(m, n, k, kind):
    x, xs, w, ws, ref = product_case(m, n, k)
    for place in range(16 // kind.itemsize):
        buf = torch.full((m * n + 64,), -7.0, dtype=kind, device="cuda")
        out = buf[16 + place:16 + place + m * n].view(m, n)
        assert L.int8_matmul(x, xs, w, ws, out=out) is out
        check_product(out, ref, kind)
        assert bool((buf[:16 + place] == -7).all()) and bool((buf[16 + place + m * n:] == -7).all())
    status_ok()


@pytest.mark.gpu
def test_product_of_weights_that_the_kernel_ahead_writes():
    """No synchronisation between what writes the operands and the product: 64 rounds with other weights each time."""
    m, n, k = 4, 8192, 2048
    x, xs, w, ws, _ = product_case(m, n, k)
    src = [int8_rows(gen(i), n, k) for i in range(4)]
    outs = []
    for i in range(64):
        w.copy_(src[i % 4])
        outs.append(L.int8_matmul(x, xs, w, ws, out_dtype="f32"))
    for i, y in enumerate(outs):
        check_product(y, x.double() @ src[i % 4].double().t() * xs.double()[:, None] * ws.double(), torch.float32)


@pytest.mark.gpu
def test_product_on_other_streams_and_threads():
    cases = [product_case(m, n, k) for m, n, k in ((1, 6000, 2048), (200, 5000, 1024), (3, 20000, 1024))]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    y = L.int8_matmul(*cases[0][:4], out_dtype="f32", stream=side)
    z = L.int8_matmul(*cases[1][:4], out_dtype="f32", stream=side.cuda_stream)
    side.synchronize()
    check_product(y, cases[0][4], torch.float32)
    check_product(z, cases[1][4], torch.float32)
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream() if i % 2 else torch.cuda.default_stream()):
            for _ in range(30):
                x, xs, w, ws, ref = cases[i % 3]
                y = L.int8_matmul(x, xs, w, ws, out_dtype="f32")
                torch.cuda.current_stream().synchronize()
                try:
                    check_product(y, ref, torch.float32)
                except AssertionError:
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong
    status_ok()


@pytest.mark.gpu
def test_graphs_do_not_share_scratch():
    """Two captured products that need scratch, replayed beside one another on two streams."""
    shapes = [(16, 9000, 4100), (300, 5000, 2001)]                         # rows off 16 bytes
    assert all(int8_matmul_workspace_bytes(*s, False, False) > int8_matmul_workspace_bytes(*s) == 0 for s in shapes)
    cases = [product_case(*s) for s in shapes]
    graphs, outs = [], []
    for c in cases:
        L.int8_matmul(*c[:4], out_dtype="f32")
    torch.cuda.synchronize()
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(L.int8_matmul(*c[:4], out_dtype="f32"))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for y in outs:
            y.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for y, c in zip(outs, cases):
            check_product(y, c[4], torch.float32)
    ws = torch.zeros(int8_matmul_workspace_bytes(*shapes[0], False, False), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = L.int8_matmul(*cases[0][:4], out_dtype="f32", workspace_buf=ws)
    g.replay()
    torch.cuda.synchronize()
    check_product(y, cases[0][4], torch.float32)
    status_ok()


@pytest.mark.gpu
def test_product_shares_scratch_with_the_int4_product():
    """One buffer a stream: the int8 product leaves the counters alone that the int4 product wants at zero."""
    x, xs, w, ws, ref = product_case(16, 9000, 4101)
    g = gen(3)
    w4 = torch.randint(0, 256, (20000, 2048), dtype=torch.uint8, device="cuda", generator=g)
    s4 = (torch.rand(20000, 128, device="cuda", generator=g) * 0.02).half()
    a = torch.randn(16, 4096, device="cuda", generator=g).half()
    torch.cuda.synchronize()
    first = L.quantized_matmul(a, w4, s4, 32)
    for _ in range(4):
        check_product(L.int8_matmul(x, xs, w, ws, out_dtype="f32"), ref, torch.float32)
        assert torch.equal(L.quantized_matmul(a, w4, s4, 32), first)
    status_ok()


@pytest.mark.gpu
def test_product_refusals():
    x, xs, w, ws, _ = product_case(4, 40, 64)
    with pytest.raises(TypeError, match="x must be int8"):
        L.int8_matmul(x.float(), xs, w, ws)
    with pytest.raises(TypeError, match="w must be int8"):
        L.int8_matmul(x, xs, w.view(torch.uint8), ws)
    with pytest.raises(ValueError, match="K="):
        L.int8_matmul(x[:, :48], xs, w, ws)
    with pytest.raises(ValueError, match="x_scales"):
        L.int8_matmul(x, xs[:3], w, ws)
    with pytest.raises(ValueError, match="x_scales"):
        L.int8_matmul(x, xs.half(), w, ws)
    with pytest.raises(ValueError, match="w_scales"):
        L.int8_matmul(x, xs, w, ws[:39])
    with pytest.raises(TypeError, match="w_scales"):
        L.int8_matmul(x, xs, w, torch.zeros(40, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="contiguous"):
        L.int8_matmul(x.t().contiguous().t(), xs, w, ws)
    with pytest.raises(ValueError, match="contiguous"):
        L.int8_matmul(x[:1].expand(4, 64), xs, w, ws)
    with pytest.raises(ValueError, match="out must hold"):
        L.int8_matmul(x, xs, w, ws, out=torch.empty(3, 40, device="cuda"))
    with pytest.raises(TypeError, match="out is"):
        L.int8_matmul(x, xs, w, ws, out=torch.empty(4, 40, device="cuda"), out_dtype="f16")
    with pytest.raises(ValueError, match="out_dtype"):
        L.int8_matmul(x, xs, w, ws, out_dtype="i8")
    with pytest.raises(ValueError, match="must be \\[K\\]"):
        L.int8_matmul(x.view(2, 2, 64), xs, w, ws)
    big = product_case(16, 5000, 1001)
    with pytest.raises(ValueError, match="workspace_buf"):
        L.int8_matmul(*big[:4], workspace_buf=torch.zeros(256, dtype=torch.uint8, device="cuda"))
    assert L.int8_matmul(x[:0], xs[:0], w, ws).shape == (0, 40)
    assert L.int8_matmul(x, xs, w[:0], ws[:0]).shape == (4, 0)
    status_ok()


# ------------------------------------------------------------------------------------------ rows
ROWS = [(1, 1), (1, 576), (5, 100), (9, 512), (2, 513), (7, 1537), (4, 4096), (33, 264), (1, 8192), (3, 8200), (2, 16384), (3, 16392), (2, 20001), (1, 50000),
        (600, 64), (1200, 1537)]


def rms(v, weight, eps=1e-5):
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * weight.double()


def check_tokens(t, v):
    """t against the row-quantised v (64 bits, itself good to REL of each row's largest value)."""
    v = v.reshape(t.scales.numel(), -1)
    amax = v.abs().amax(-1, keepdim=True)
    s = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
    assert bool(((t.scales.reshape(-1, 1).double() - s).abs() <= 2 * REL * s).all())
    quotient, q = v / s, t.q.reshape(v.shape).double()
    assert bool(((q - quotient).abs() <= 0.5 + 127 * 2 * REL).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,n", ROWS)
def test_rows_against_64_bits(rows, n, kind):
    g = gen(rows, n)

    def draw(r, scale=1.0, plus=0.0):
        return (torch.randn(r, n, device="cuda", generator=g) * scale + plus).to(kind)
    x, delta, w, post = draw(rows), draw(rows, 3.0), draw(1, 0.1, 1.0)[0], draw(1, 0.1, 1.0)[0]
    t = L.quantize_tokens(x)
    assert t.q.shape == x.shape and t.scales.shape == (rows,) and (t.q.stride(0) % 16 == 0 or rows == 1)
    whole = L.quantize(x, n, bits=8)                                     # bit for bit the weight quantiser's
    assert torch.equal(t.q, whole.w) and torch.equal(t.scales, whole.scales.view(-1))
    check_tokens(L.quantize_tokens(x, w), rms(x.double(), w))
    gu = torch.randn(rows, 2 * n, device="cuda", generator=g).to(kind)
    a, b = gu[:, :n].double(), gu[:, n:].double()
    check_tokens(L.silu_mul_tokens(gu[:, :n], gu[:, n:]), a * torch.sigmoid(a) * b)
    for has_post, gate_rows, scale in ((True, 1, 0.5), (False, rows, -1.5), (True, 0, 1.0), (False, 0, 1.0)):
        gate = draw(gate_rows, 0.5) if gate_rows else None
        y = rms(delta.double(), post) if has_post else delta.double()
        if gate_rows:
            y = y * gate.double()
        y = scale * y
        ref = x.double() + y
        hidden = torch.empty_like(x)
        out = L.residual_norms(x, delta, w, gate=gate, post_weight=post if has_post else None, scale=scale, hidden_out=hidden)
        slack = REL * y.abs() + 2.0 ** -24 * ref.abs()
        assert bool(((hidden.double() - ref).abs() <= HALF_STEP[kind] * ref.abs() + (1 + HALF_STEP[kind]) * slack + 2.0 ** -25).all())
        normed = rms(hidden.double(), w)
        assert bool(((out.double() - normed).abs() <= (HALF_STEP[kind] + 1.01 * REL) * normed.abs() + 2.0 ** -25).all())
        again = x.clone()
        tokens = L.residual_norms(again, delta, w, gate=gate, post_weight=post if has_post else None, scale=scale, quantized=True)
        assert torch.equal(again, hidden)                                # in place and beside give the same
        check_tokens(tokens, normed)
        once = x.clone()
        assert L.residual_norms(once, delta, gate=gate, post_weight=post if has_post else None, scale=scale) is once and torch.equal(once, hidden)
    plain, ours = x.clone(), x.clone()                                   # the case that the package had before
    a, b = L.residual_rms_norm(plain, delta, w), L.residual_norms(ours, delta, w)
    assert torch.equal(plain, ours)
    assert bool(((a.double() - b.double()).abs() <= 2 * (HALF_STEP[kind] + REL) * a.double().abs() + 2.0 ** -24).all())
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [64, 65, 1024, 9000])
def test_a_gate_row_serves_its_sequence(n):
    g = gen(n)
    x, d = (torch.randn(12, n, device="cuda", generator=g) for _ in range(2))
    gate = torch.randn(3, n, device="cuda", generator=g)
    out = x.clone()
    L.residual_norms(out, d, gate=gate)
    assert bool(((out - (x + d * gate.repeat_interleave(4, 0))).abs() <= 1e-6 * (x.abs() + (d * gate.repeat_interleave(4, 0)).abs())).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 41, 600, 20000])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_hold_no_number(kind, n):
    """Zeros, infinities, NaN, the type's lowest and smallest values: each stays in its row."""
    g = gen(n)
    x = torch.randn(8, n, device="cuda", generator=g).to(kind)
    x[0] = 0
    x[1, n // 2], x[2, 3], x[3, n - 1] = float("nan"), float("inf"), float("-inf")
    x[4] = torch.finfo(kind).min
    x[5] = torch.finfo(kind).smallest_normal * 2.0 ** -4                 # subnormal in the type
    w = torch.ones(n, device="cuda", dtype=kind)
    t = L.quantize_tokens(x)
    assert bool((t.q[:4] == 0).all()) and t.scales[0] == 1 and bool(t.scales[1:4].isnan().all())
    assert bool((t.q[4] == -127).all())
    assert torch.allclose(t.scales[4].double(), torch.tensor(-torch.finfo(kind).min / 127).double().cuda(), rtol=1e-6)
    assert t.scales[5] >= 2.0 ** -126 and bool((t.q[5] >= 0).all())
    v5 = t.q[5].double() * t.scales[5].double()
    assert bool(((v5 - x[5].double()).abs() <= 0.5 * t.scales[5].double()).all())
    check_tokens(L.QuantizedTokens(t.q[6:], t.scales[6:]), x[6:].double())
    t = L.quantize_tokens(x, w)
    assert bool((t.q[:4] == 0).all()) and t.scales[0] == 1 and bool(t.scales[1:4].isnan().all())
    check_tokens(L.QuantizedTokens(t.q[6:], t.scales[6:]), rms(x[6:].double(), w))
    out = L.residual_norms(torch.zeros_like(x), x, w)
    assert bool((out[0] == 0).all()) and bool(out[1].isnan().all()) and bool((out[2, :3] == 0).all()) and bool(out[2, 3].isnan())
    q = L.residual_norms(torch.zeros_like(x), x, w, post_weight=w, quantized=True)
    assert q.scales[0] == 1 and bool(q.scales[1:4].isnan().all()) and bool(q.scales[6:].isfinite().all())
    gu = L.silu_mul_tokens(x, torch.ones_like(x))
    assert bool(gu.scales[1:3].isnan().all()) and bool(gu.scales[6:].isfinite().all())
    weights = L.quantize(torch.randn(16, n, device="cuda", generator=g), n, bits=8)
    y = L.int8_matmul(L.quantize_tokens(x).q, L.quantize_tokens(x).scales, weights.w, weights.scales, out_dtype="f32")
    assert bool(y[1:4].isnan().all()) and bool((y[0] == 0).all()) and bool(y[6:].isfinite().all())


@pytest.mark.gpu
def test_rows_of_views_and_odd_addresses():
    g = gen(5)
    for kind in KINDS:
        wide = torch.randn(9, 700, device="cuda", generator=g).to(kind)
        for start, n in ((0, 512), (8, 512), (3, 512), (1, 333), (0, 600)):
            x = wide[:, start:start + n]
            a, b = L.quantize_tokens(x), L.quantize_tokens(x.contiguous())
            assert torch.equal(a.q, b.q) and torch.equal(a.scales, b.scales)
            up = wide.flip(0)[:, start:start + n]
            a, b = L.silu_mul_tokens(x, up), L.silu_mul_tokens(x.contiguous(), up.contiguous())
            assert torch.equal(a.q, b.q) and torch.equal(a.scales, b.scales)
        flat = torch.randn(4 * 96 + 1, device="cuda", generator=g).to(kind)
        x = flat[1:].view(4, 96)                                          # contiguous, off 16 bytes
        w = torch.ones(96, device="cuda", dtype=kind)
        assert torch.equal(L.residual_norms(x.clone(), x, w), L.residual_norms(x.clone(), x.clone(), w))
        three = torch.randn(2, 3, 40, device="cuda", generator=g).to(kind)
        t = L.quantize_tokens(three)
        assert t.q.shape == (2, 3, 40) and t.scales.shape == (2, 3) and torch.equal(t.q.reshape(6, 40), L.quantize_tokens(three.view(6, 40)).q)
        one = L.quantize_tokens(three[0, 0])
        assert one.q.shape == (40,) and one.scales.shape == () and torch.equal(one.q, t.q[0, 0])


@pytest.mark.gpu
def test_rows_write_their_rows_and_nothing_else():
    g = gen(6)
    for n, ld in ((100, 112), (512, 512), (333, 400), (64, 80)):
        x = torch.randn(6, n, device="cuda", generator=g).half()
        q = torch.full((8, ld), 99, dtype=torch.int8, device="cuda")
        s = torch.full((8,), 9.0, device="cuda")
        t = L.QuantizedTokens(q[1:7, :n], s[1:7])
        assert L.quantize_tokens(x, out=t) is t
        want = L.quantize_tokens(x)
        assert torch.equal(t.q, want.q) and torch.equal(t.scales, want.scales)
        assert bool((q[0] == 99).all()) and bool((q[7] == 99).all()) and bool((q[:, n:] == 99).all()) and s[0] == 9 and s[7] == 9
        h = x.clone()
        assert L.residual_norms(h, x, torch.ones(n, device="cuda").half(), quantized=True, out=t) is t
        d = x.clone()
        assert L.residual_norms(x.clone(), d, torch.ones(n, device="cuda").half(), out=d) is d           # out may be delta
        assert torch.equal(d, L.residual_norms(x.clone(), x, torch.ones(n, device="cuda").half()))


@pytest.mark.gpu
def test_general_path_gives_the_same_bits():
    g = gen(7)
    D = L.DeviceTensor
    x, d = (torch.randn(5, 192, device="cuda", generator=g).half() for _ in range(2))
    w, gate = (torch.randn(192, device="cuda", generator=g).half() for _ in range(2))

    def same(a, b):
        return torch.equal(a.q, b.q) and torch.equal(a.scales, b.scales)
    assert same(L.quantize_tokens(x, w), L.quantize_tokens(D(x), w)) and same(L.quantize_tokens(x), L.quantize_tokens(x.cpu().numpy()))
    assert same(L.silu_mul_tokens(x, d), L.silu_mul_tokens(D(x), d))
    a, b = x.clone(), x.clone()
    assert torch.equal(L.residual_norms(a, d, w, 1e-6, post_weight=gate, gate=gate, scale=0.25),
                       L.residual_norms(D(b), d, w, 1e-6, post_weight=gate, gate=gate, scale=0.25)) and torch.equal(a, b)
    host = torch.empty(5, 192, dtype=torch.float16).numpy()
    assert L.residual_norms(D(x.clone()), d, w, out=host) is host and torch.equal(torch.from_numpy(host).cuda(), L.residual_norms(x.clone(), d, w))
    c = L.residual_norms(x.view(torch.float16), d, w, bf16=True, hidden_out=torch.empty_like(x))           # bits of bfloat16 in a float16 array
    assert torch.equal(c.view(torch.bfloat16) if c.dtype == torch.float16 else c,
                       L.residual_norms(x.view(torch.bfloat16).clone(), d.view(torch.bfloat16), w.view(torch.bfloat16)))
    t, weights = L.quantize_tokens(x), L.quantize(torch.randn(40, 192, device="cuda", generator=g), 192, bits=8)
    y = L.int8_matmul(t.q, t.scales, weights.w, weights.scales)
    assert torch.equal(y, L.int8_matmul(D(t.q), t.scales, weights.w, weights.scales))
    host = torch.empty(5, 40, dtype=torch.float16).numpy()
    assert L.int8_matmul(t.q, t.scales, weights.w, weights.scales, out=host) is host and torch.equal(torch.from_numpy(host).cuda(), y)


@pytest.mark.gpu
def test_row_refusals():
    x = torch.randn(6, 64, device="cuda").half()
    w = torch.ones(64, device="cuda").half()
    with pytest.raises(ValueError, match="weight must hold"):
        L.quantize_tokens(x, w[:63])
    with pytest.raises(TypeError, match="one dtype"):
        L.quantize_tokens(x, w.float())
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        L.quantize_tokens(x.to(torch.int8))
    with pytest.raises(ValueError, match="contiguous"):
        L.quantize_tokens(x.t())
    with pytest.raises(ValueError, match="contiguous"):
        L.quantize_tokens(x[:1].expand(6, 64))
    with pytest.raises(ValueError, match="out.q"):
        L.quantize_tokens(x, out=L.QuantizedTokens(torch.empty(5, 64, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")))
    with pytest.raises(ValueError, match="out.scales"):
        L.quantize_tokens(x, out=L.QuantizedTokens(torch.empty(6, 64, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")))
    with pytest.raises(TypeError, match="QuantizedTokens"):
        L.residual_norms(x, x, w, quantized=True, out=torch.empty_like(x))
    with pytest.raises(ValueError, match="one shape"):
        L.silu_mul_tokens(x, x[:3])
    with pytest.raises(ValueError, match="delta"):
        L.residual_norms(x, x[:3], w)
    with pytest.raises(ValueError, match="gate"):
        L.residual_norms(x, x, w, gate=torch.ones(4, 64, device="cuda").half())
    with pytest.raises(ValueError, match="gate"):
        L.residual_norms(x, x, w, gate=w[:32])
    with pytest.raises(ValueError, match="without weight"):
        L.residual_norms(x, x, quantized=True)
    with pytest.raises(ValueError, match="without weight"):
        L.residual_norms(x, x, out=torch.empty_like(x))
    with pytest.raises(ValueError, match="hidden_out"):
        L.residual_norms(x, x, w, hidden_out=torch.empty(5, 64, device="cuda").half())
    with pytest.raises(TypeError, match="in place"):
        L.residual_norms(x.cpu().numpy(), x, w)
    with pytest.raises(ValueError, match="normalised"):
        L.Int8Linear(torch.zeros(8, 64, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda"))(L.quantize_tokens(x), w)
    empty = L.quantize_tokens(x[:0])
    assert empty.q.shape == (0, 64) and empty.scales.shape == (0,)
    status_ok()


@pytest.mark.gpu
def test_tokens_into_other_objects():
    """Outputs given as this package's tensors; the general path writes where the native one does."""
    x = torch.randn(6, 100, device="cuda", generator=gen(9)).half()
    q, s = L.empty((6, 112), dtype="int8"), L.empty(6)
    want = L.quantize_tokens(x)
    with pytest.raises(ValueError, match="out.q"):
        L.quantize_tokens(x, out=L.QuantizedTokens(q, s))                 # rows of 112
    t = L.QuantizedTokens(L.DeviceTensor(torch.empty(6, 100, dtype=torch.int8, device="cuda")), s)
    assert L.quantize_tokens(x, out=t) is t and torch.equal(t.q.torch(), want.q) and torch.equal(s.torch(), want.scales)
    assert L.silu_mul_tokens(x, x, out=t) is t and torch.equal(t.q.torch(), L.silu_mul_tokens(x, x).q)
    w = torch.ones(100, device="cuda").half()
    assert L.residual_norms(x.clone(), x, w, quantized=True, out=t) is t
    with pytest.raises(TypeError, match="device"):
        L.quantize_tokens(x, out=L.QuantizedTokens(want.q.cpu().numpy().copy(), s))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows, weights and outputs of more than 2^31 values: the last ones are where they belong."""
    n, rows = 32768, 66000                                                # 2.16e9 values
    x = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    x[:] = torch.randn(1, n, device="cuda", generator=gen(10))
    x[-3:] *= torch.tensor([[2.0], [0.0], [3.0]], device="cuda", dtype=torch.bfloat16)
    t = L.quantize_tokens(x)
    small = L.quantize_tokens(x[-4:].contiguous())
    assert torch.equal(t.q[-4:], small.q) and torch.equal(t.scales[-4:], small.scales) and torch.equal(t.q[0], t.q[rows // 2])
    w = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(x)
    L.residual_norms(x, x, w, hidden_out=out, out=out)                    # (out twice: the norm is what stays)
    h = x[-4:].float() + x[-4:].float()
    ref = L.rms_norm(h.to(torch.bfloat16), w)
    assert bool(((out[-4:].double() - ref.double()).abs() <= 2.0 ** -7 * ref.double().abs()).all())
    del out, x
    k = 64
    a, xs, b, ws, _ = product_case(rows, n, k)
    y = L.int8_matmul(a, xs, b, ws)                                       # 2.16e9 outputs
    check_product(y[-5:], a[-5:].double() @ b.double().t() * xs[-5:].double()[:, None] * ws.double(), torch.float16)
    check_product(y[:5], a[:5].double() @ b.double().t() * xs[:5].double()[:, None] * ws.double(), torch.float16)
    del y
    wide = torch.randint(-128, 128, (300000, 8192), dtype=torch.int8, device="cuda", generator=gen(11))          # 2.46e9 weights
    scales = torch.rand(300000, device="cuda", generator=gen(12)) * 0.01
    for m in (1, 5, 16, 70):
        x8, xs, _, _, _ = product_case(m, 8, 8192)
        y = L.int8_matmul(x8, xs, wide, scales, out_dtype="f32")
        check_product(y[:, -300:], x8.double() @ wide[-300:].double().t() * xs.double()[:, None] * scales[-300:].double(), torch.float32)
    odd = wide.view(-1)[:300000 * 8191].view(300000, 8191)                # rows off 16 bytes, 51 pieces
    y = L.int8_matmul(x8[:, :8191], xs, odd, scales, out_dtype="f32")
    check_product(y[:, -300:], x8[:, :8191].double() @ odd[-300:].double().t() * xs.double()[:, None] * scales[-300:].double(), torch.float32)
    y = L.int8_matmul(x8[:3, :8191], xs[:3], odd, scales, out_dtype="f32")
    check_product(y[:, -300:], x8[:3, :8191].double() @ odd[-300:].double().t() * xs[:3].double()[:, None] * scales[-300:].double(), torch.float32)
    status_ok()


# ------------------------------------------------------------------------------------------ together
@pytest.mark.gpu
@pytest.mark.parametrize("m,hidden,inter", [(1, 576, 1536), (5, 200, 333), (16, 512, 1024), (130, 264, 700)])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
def test_an_mlp_block(m, hidden, inter, kind):
    """Norm, gate and up, SiLU, down, norm after, residual, norm before the next: each step against 64 bits on what the step before
    gave, the layers' forms among each other, and the whole in a graph."""
    g = gen(m, hidden, inter)

    def draw(*shape, plus=0.0, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale + plus).to(kind)
    x, w_in, w_post, w_next = draw(m, hidden), draw(hidden, plus=1.0, scale=0.1), draw(hidden, plus=1.0, scale=0.1), draw(hidden, plus=1.0, scale=0.1)
    up = L.quantize(torch.randn(2 * inter, hidden, device="cuda", generator=g), hidden, bits=8)
    down = L.quantize(torch.randn(hidden, inter, device="cuda", generator=g), inter, bits=8)
    up_layer, down_layer = up.int8_linear(), down.int8_linear()

    def block(stream_hidden):
        gu = up_layer(x, w_in, out_dtype="f16")
        d = down_layer(L.silu_mul_tokens(gu[:, :inter], gu[:, inter:]), out_dtype=NAMES[kind])
        return gu, d, L.residual_norms(stream_hidden, d, w_next, post_weight=w_post, scale=0.5, quantized=True)
    h = x.clone()
    gu, d, tokens = block(h)
    t = L.quantize_tokens(x, w_in)
    check_tokens(t, rms(x.double(), w_in))

    def product(t, q):
        return t.q.double() @ q.w.double().t() * t.scales.double()[:, None] * q.scales.double().view(-1)
    check_product(gu, product(t, up), torch.float16)
    assert torch.equal(gu, L.int8_matmul(t.q, t.scales, up.w, up.scales))
    t = L.silu_mul_tokens(gu[:, :inter], gu[:, inter:])
    a, b = gu[:, :inter].double(), gu[:, inter:].double()
    check_tokens(t, a * torch.sigmoid(a) * b)
    check_product(d, product(t, down), kind)
    ref = x.double() + 0.5 * rms(d.double(), w_post)
    assert bool(((h.double() - ref).abs() <= (HALF_STEP[kind] + 2 * REL) * (ref.abs() + x.double().abs())).all())
    check_tokens(tokens, rms(h.double(), w_next))
    graph = torch.cuda.CUDAGraph()
    h2 = x.clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        h2.copy_(x)
        _, _, tokens2 = block(h2)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(h2, h) and torch.equal(tokens2.q, tokens.q) and torch.equal(tokens2.scales, tokens.scales)
    status_ok()


@pytest.mark.gpu
def test_layer_forms():
    g = gen(8)
    for n, k in ((100, 333), (64, 512)):
        q = L.quantize(torch.randn(n, k, device="cuda", generator=g), k, bits=8)
        layer = q.int8_linear()
        assert layer.w.stride(0) % 16 == 0 and layer.weight_bytes == n * k + 4 * n
        for kind in KINDS:
            x = torch.randn(7, k, device="cuda", generator=g).to(kind)
            y = layer(x)
            assert y.dtype == kind and y.shape == (7, n)
            t = L.quantize_tokens(x)
            assert torch.equal(layer(t, out_dtype=NAMES[kind]), y) and torch.equal(layer(x[3]), y[3])
            out = torch.empty_like(y)
            assert layer(x, out=out) is out and torch.equal(out, y)
            err = (y.double() - x.double() @ (q.w.double() * q.scales.double()).t()).norm() / y.double().norm()
            assert err < 0.02
    with pytest.raises(ValueError, match="one scale"):
        L.quantize(torch.randn(8, 64, device="cuda"), 32, bits=8).int8_linear()
    with pytest.raises(ValueError, match="one scale"):
        L.quantize(torch.randn(8, 64, device="cuda"), 64, bits=4).int8_linear()


@pytest.mark.gpu
def test_rows_on_another_stream():
    x = torch.randn(64, 4096, device="cuda").half()
    w = torch.ones(4096, device="cuda").half()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    a = L.quantize_tokens(x, w, stream=side)
    h = x.clone()
    torch.cuda.synchronize()
    n = L.residual_norms(h, x, w, stream=side)
    s = L.silu_mul_tokens(x, x, stream=side)
    side.synchronize()
    b = L.quantize_tokens(x, w)
    assert torch.equal(a.q, b.q) and torch.equal(n, L.residual_norms(x.clone(), x, w)) and torch.equal(s.q, L.silu_mul_tokens(x, x).q)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("post_norms,scale", [(False, 1.0), (True, 0.5)])
def test_decode_stack_in_int8(kind, post_norms, scale):
    """Every launch of two layers against 64 bits on what the launches before it left, and the same step from a graph."""
    st = L.DecodeStack(layers=2, hidden=200, inter=333, q_heads=3, kv_heads=1, head_dim=40, vocab=1000, fused=True, glue=True, int8=True, dtype=kind,
                       post_norms=post_norms, residual_scale=scale, seed=4)
    assert st.launches_per_step == len(st.ops) == 2 + 7 * 2 + 2
    st.token.fill_(77)
    for t in (st.normed, st.mlp):
        t.q.zero_()
    ops, norms, calls = iter(st.ops), iter(st.norms), iter(st.calls)

    def linear():
        lin, tokens, out = next(calls)
        next(ops)()
        ref = tokens.q.double() @ lin.w.double().t() * tokens.scales.double()[:, None] * lin.scales.double()
        check_product(out, ref, kind)
        return out

    def block_end(delta):
        before = st.hidden.double()
        next(ops)()
        y = rms(delta.double(), next(norms)) if post_norms else delta.double()
        ref = before + scale * y
        assert bool(((st.hidden.double() - ref).abs() <= (HALF_STEP[kind] + 2 * REL) * (ref.abs() + before.abs()) + 2.0 ** -25).all())
        check_tokens(st.normed, rms(st.hidden.double(), next(norms)))
    next(ops)()
    assert torch.equal(st.hidden[0], st.table[77])
    next(ops)()
    check_tokens(st.normed, rms(st.hidden.double(), next(norms)))
    for _ in range(2):
        linear()
        block_end(linear())
        gu = linear()
        next(ops)()
        a, b = gu[:, :333].double(), gu[:, 333:].double()
        check_tokens(st.mlp, a * torch.sigmoid(a) * b)
        block_end(linear())
    logits = linear()
    next(ops)()
    assert int(st.next_token) == int(logits.float().argmax()) and not list(ops) and not list(norms)
    want, token = logits.clone(), int(st.next_token)
    st.capture()
    logits.zero_()
    st.next_token.zero_()
    st.replay()
    torch.cuda.synchronize()
    assert torch.equal(st.logits, want) and int(st.next_token) == token
    status_ok()


def test_decode_stack_says_what_int8_needs():
    with pytest.raises(ValueError, match="glue"):
        L.DecodeStack(layers=1, fused=True, int8=True, device="cpu")
    with pytest.raises(ValueError, match="int8 form"):
        L.DecodeStack(layers=1, fused=True, glue=True, post_norms=True, device="cpu")
