"""GPU: Int8Linear against the same product in 64 bits.

The codes and the integer sum are exact, so what remains are the conversions of the
sum and of the scales' product to fp32 and their product (three roundings, below
2^-22) and the rounding to the output's type (half an ulp: 2^-9 in bf16, 2^-12 in
fp16, doubled for the binade's edge; below fp16's normal range 2^-25 absolutely).
"""
import ctypes

import pytest
import torch

import megaqwen_b200 as mq
from megaqwen_b200 import _lib

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rand(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _weights(n, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8),
            torch.rand(n, generator=g, device="cuda") * 1e-2 + 1e-4)


def reference(x, w, s):
    """(codes c W^T) s_x s_w in float64; the codes as the definition has them, with fp32 divisions."""
    x = x.cpu().float().reshape(-1, x.shape[-1])
    sx = (x.abs().amax(-1, keepdim=True) / 127).clamp_min(1e-12)
    c = torch.round(x / sx)
    return ((c.cuda().double() @ w.double().t()) * sx.cuda().double() * s.double()).cpu()


def check(y, ref):
    ulp = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}[y.dtype]
    y = y.cpu().double().reshape(ref.shape)
    bound = (ulp + 2.0 ** -22) * ref.abs() + (2.0 ** -24 if ulp == 2.0 ** -11 else 1e-40)
    assert torch.isfinite(y).all() and float(((y - ref).abs() / bound).max()) <= 1.0


# tokens: the few-token kernel (1..4), every tile width and its edges, several tiles; odd rows, channels and K
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 16, 17, 33, 64, 65, 128, 129, 257, 300, 513])
@pytest.mark.parametrize("n,k", [(1, 1), (31, 17), (128, 128), (129, 127), (300, 1000), (1024, 2048), (40, 4095)])
def test_shapes(m, n, k):
    w, s = _weights(n, k, n + k)
    x = _rand((m, k), m)
    lin = mq.Int8Linear(w, s)
    check(lin(x, out_dtype=torch.float32), reference(x, w, s))
    lin.check_device()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("m", [1, 3, 40, 200])
def test_types(dtype, out, m):
    w, s = _weights(515, 333, 5)
    s *= 0.01
    x = _rand((m, 333), m, dtype)
    check(mq.Int8Linear(w, s)(x, out_dtype=out), reference(x, w, s))
    assert mq.Int8Linear(w, s)(x).dtype == dtype


@pytest.mark.parametrize("m,n,k", [(1, 4096, 1024), (4, 6144, 1024), (7, 1024, 2048), (64, 20000, 1024), (1000, 4096, 1024),
                                   (2500, 640, 512), (2, 64, 30000), (9, 64, 30000), (1, 16, 100000), (40, 128, 131072)])
def test_larger(m, n, k):
    """The model's projections, many tiles for each CTA, and long sums (the few-token kernel ends at 65,536 codes)."""
    w, s = _weights(n, k, 3)
    x = _rand((m, k), 4)
    lin = mq.Int8Linear(w, s)
    check(lin(x, out_dtype=torch.float32), reference(x, w, s))
    lin.check_device()


@pytest.mark.parametrize("m,n,k", [(2500, 2048, 256), (4737, 1024, 130), (1300, 4091, 96), (129, 20001, 64), (5000, 1288, 17)])
@pytest.mark.parametrize("out", TYPES)
def test_enough_tiles_for_every_sm(m, n, k, out):
    """Tokens as the rows of the tensor-core tiles: ragged last tiles in both directions, rows of y that are 16-byte
    aligned (they leave by TMA) and rows that are not."""
    w, s = _weights(n, k, 7)
    s *= 0.01
    x = _rand((m, k), 8)
    lin = mq.Int8Linear(w, s)
    y = lin(x, out_dtype=out)
    check(y, reference(x, w, s))
    lin.check_device()


def test_largest_sums():
    """Every code at its extreme: the int32 sum comes within 1 % of its range, and does not wrap."""
    for m in (1, 40):
        k = 131072
        w = torch.full((16, k), -128, dtype=torch.int8, device="cuda")
        x = torch.ones((m, k), device="cuda") if m == 40 else torch.ones((m, 65536), device="cuda")
        w = w[:, :x.shape[1]].contiguous()
        s = torch.ones(16, device="cuda")
        check(mq.Int8Linear(w, s)(x), reference(x, w, s))


@pytest.mark.parametrize("m", [1, 3, 20])
def test_edges_of_the_quantiser(m):
    """Ties, zeros, tiny and huge tokens; a token with an infinity or a NaN gives NaN and leaves the others alone."""
    k, n = 130, 70
    w, s = _weights(n, k, 1)
    rows = torch.zeros((8, k), device="cuda")
    rows[0, :100] = torch.arange(100, device="cuda") - 49.5     # scale 1: half-way values
    rows[0, 100] = 127.0
    rows[2] = 1e-30
    rows[3, 0] = 3e38
    rows[4] = _rand((k,), 1, torch.float32) * 1e-13
    rows[5] = _rand((k,), 2, torch.float32) * 1e20
    rows[6, 129] = -1.0
    s *= 1e-3
    lin = mq.Int8Linear(w, s)
    for i in range(8):
        x = _rand((m, k), 9, torch.float32)
        x[m - 1] = rows[i]
        check(lin(x), reference(x, w, s))
    for bad in (float("inf"), float("nan"), -float("inf")):
        x = _rand((m, k), 9, torch.float32)
        ref = reference(x, w, s)
        x[m - 1, k - 1] = bad
        y = lin(x)
        assert y[m - 1].isnan().all()
        if m > 1:
            check(y[:m - 1], ref[:m - 1])


@pytest.mark.parametrize("m", [2, 30])
def test_strides_alignment_and_shapes(m):
    """Views of wider rows, at offsets without 16-byte alignment; weights that are columns of a wider matrix, whose
    neighbours must not count; leading axes; another stream."""
    k, n = 100, 60
    wide_w, s = _weights(n, 256, 1)
    for woff in (0, 16, 3):
        w = wide_w[:, woff:woff + k]
        for wk in (k, 96):
            lin = mq.Int8Linear(w[:, :wk], s)
            for xoff in (0, 1, 8):
                x = _rand((m, 3 * k), 2)[:, xoff:xoff + wk]
                check(lin(x, out_dtype=torch.float32), reference(x, w[:, :wk], s))
    lin = mq.Int8Linear(wide_w[:, :96], s)
    x = _rand((2, m, 1, 96), 3)
    y = lin(x, out_dtype=torch.float32)
    assert y.shape == (2, m, 1, n)
    check(y, reference(x, wide_w[:, :96], s))
    tr = _rand((m, 2, 96), 4).transpose(0, 1)
    check(lin(tr, out_dtype=torch.float32), reference(tr, wide_w[:, :96], s))
    assert lin(x[:, :0]).shape == (2, 0, 1, n)
    assert lin(_rand((96,), 5)).shape == (n,)
    ref = reference(x, wide_w[:, :96], s)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        there = [lin(x, out_dtype=torch.float32) for _ in range(5)]
    here = [lin(x, out_dtype=torch.float32) for _ in range(5)]
    torch.cuda.synchronize()
    for y in there + here:
        check(y, ref)


def test_many_calls_in_a_row():
    """Back-to-back calls of different widths share the workspace, and each sees its own codes."""
    layers = [(mq.Int8Linear(w, s), w, s) for w, s in (_weights(n, 512, n) for n in (64, 700, 2000))]
    xs = [_rand((m, 512), m) for m in (1, 6, 20, 70, 130, 600)]
    for _ in range(3):
        ys = [(l(x, out_dtype=torch.float32), x, w, s) for x in xs for l, w, s in layers]
    for y, x, w, s in ys:
        check(y, reference(x, w, s))


def test_weights_of_the_quantiser():
    """quantize_per_channel's weights and a bf16 activation: close to the bf16 product itself."""
    w = _rand((512, 1024), 1)
    x = _rand((33, 1024), 2)
    y = mq.Int8Linear(*mq.quantize_per_channel(w))(x, out_dtype=torch.float32).cpu().double()
    ref = x.cpu().double() @ w.cpu().double().t()
    assert float((y - ref).norm() / ref.norm()) < 0.02     # two roundings to 8 bits, uniform within a step of max/127


def test_refusals():
    w, s = _weights(32, 64, 1)
    for bad in ((w.cpu(), s), (w.float(), s), (w[0], s), (w, s[:5]), (w, s.half()), (w, s.cpu()), (w[:0], s[:0])):
        with pytest.raises(ValueError):
            mq.Int8Linear(*bad)
    with pytest.raises(TypeError):
        mq.Int8Linear([[1]], s)
    with pytest.raises(ValueError):
        mq.Int8Linear(torch.zeros((1, 131073), dtype=torch.int8, device="cuda"), s[:1])
    lin = mq.Int8Linear(w, s)
    x = _rand((4, 64), 1)
    for bad in (x.cpu(), x.double(), x[:, :63], _rand((64, 4), 1).t()):
        with pytest.raises(ValueError):
            lin(bad)
    with pytest.raises(ValueError):
        lin(x, out_dtype=torch.float64)
    with pytest.raises(TypeError):
        lin(None)


def test_c_entry_point_refuses():
    lib = _lib.load()
    w, s = _weights(32, 64, 1)
    x, y = _rand((8, 64), 1), torch.empty((8, 32), device="cuda")
    st = torch.zeros(2, dtype=torch.int32, device="cuda")
    nb = ctypes.c_size_t(0)
    assert lib.mq_linear8_workspace_bytes(8, 64, ctypes.byref(nb)) == 0 and nb.value
    assert lib.mq_linear8_workspace_bytes(8, 0, ctypes.byref(nb)) == -1
    lib.mq_linear8_workspace_bytes(8, 64, ctypes.byref(nb))
    ws = torch.empty(nb.value, dtype=torch.uint8, device="cuda")
    good = dict(x=x.data_ptr(), dt=0, xs=64, w=w.data_ptr(), ldw=64, s=s.data_ptr(), y=y.data_ptr(), od=2, m=8, n=32, k=64,
                ws=ws.data_ptr(), nb=nb.value, st=st.data_ptr(), stream=None)
    call = lambda **kw: lib.mq_linear8(*{**good, **kw}.values())
    assert call() == 0
    for kw in ({"x": None}, {"w": None}, {"s": None}, {"y": None}, {"st": None}, {"dt": 3}, {"od": -1}, {"m": -1}, {"n": 0},
               {"k": 0}, {"ldw": 56}, {"ldw": 48}, {"w": w.data_ptr() + 8}, {"x": x.data_ptr() + 1}, {"xs": -64}):
        assert call(**kw) == -1, kw
    for kw in ({"nb": nb.value - 64}, {"ws": None}, {"k": 131073, "ldw": 131088}):
        assert call(**kw) == -5, kw
    assert call(m=0, x=None) == 0
    torch.cuda.synchronize()


# few tokens on both sides of the rule between the one kernel and the two, and rows that are not 16-byte aligned
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 40000, 833), (1, 41000, 833), (2, 20000, 835), (2, 21000, 835), (3, 700, 2729), (3, 700, 2733),
                                   (4, 900, 2048), (4, 900, 2049)])
def test_few_tokens(m, n, k, dtype):
    w, s = _weights(n, k, n + k)
    x = _rand((m, k), m, dtype)
    check(mq.Int8Linear(w, s)(x, out_dtype=torch.float32), reference(x, w, s))


def test_captured_calls_keep_their_workspace():
    """A graph's calls give the eager results after the stream has seen larger calls, and beside them."""
    w, s = _weights(700, 512, 3)
    lin = mq.Int8Linear(w, s)
    x, big = _rand((40, 512), 1), _rand((3000, 512), 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want, want_big = lin(x), lin(big)
        lin(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = lin(x)
        beside = [lin(big) for _ in range(4)]
    for _ in range(4):
        graph.replay()                 # on the current stream, while `side` may still run
    torch.cuda.synchronize()
    assert torch.equal(y, want) and all(torch.equal(b, want_big) for b in beside)


# M * K = 8192 codes are the most that the kernel for few tokens takes; one 16-byte unit more goes to the tensor cores
@pytest.mark.parametrize("m,k", [(1, 8192), (2, 4096), (4, 2048), (1, 8208), (4, 2064)])
def test_largest_sums_of_few_tokens(m, k):
    """All codes at their extremes, on both sides of the rule between the kernels; signs that alternate in the second row."""
    s = torch.ones(16, device="cuda")
    for value in (-128, 127):
        w = torch.full((16, k), value, dtype=torch.int8, device="cuda")
        x = torch.ones((m, k), device="cuda")
        x[m - 1, 1::2] = -1.0 if m > 1 else 1.0
        check(mq.Int8Linear(w, s)(x), reference(x, w, s))
