"""Every kernel of the FP8 product, exactly; the operators' native entries against their general ones; workspaces,
graphs and buffers that are shared."""

import ctypes
import threading

import pytest
import torch

from fp8_util import U, check_product, check_quant, make_rows, make_weight, norm64, weight64
from sglang_exl3 import _lib, ops

pytestmark = pytest.mark.gpu
BF, HF, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _registered():
    ops.register_custom_ops()


def op():
    return torch.ops.sglang_exl3


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


# One shape or more for each kernel, tile and way to split k that sizes lead to.
SHAPES = [
    # the weight streamed by 2, 4 and 8 waves
    (1, 128, 16), (1, 1024, 16), (1, 11008, 16), (600, 11008, 16), (16, 1024, 8192), (3, 4096, 2048),
    # rings of 16 .. 128 rows and 64 columns, k whole and split
    (17, 5120, 16), (12, 5120, 16), (128, 512, 2048), (12, 1024, 14336), (129, 7168, 16), (17, 5120, 4096),
    (256, 128, 1536), (17, 128, 14336), (257, 7168, 16), (33, 5120, 4096), (384, 128, 1024), (33, 128, 10240),
    (400, 11008, 16), (50, 4096, 5120), (400, 128, 1024), (50, 128, 14336), (600, 28672, 16), (768, 128, 512),
    (65, 128, 14336),
    # and 128 columns
    (100, 5120, 1536), (65, 640, 6144), (5, 128, 28672), (150, 11008, 1536), (129, 128, 6144), (17, 128, 28672),
    (384, 11008, 1024), (257, 256, 4096), (33, 128, 28672), (400, 4096, 1536), (50, 11008, 6144), (257, 128, 6144),
    (50, 128, 28672), (600, 7168, 4096), (257, 128, 8192), (65, 128, 28672),
    # tiles of 256 x 256: whole ones, halves of them, 128 last rows
    (8192, 7168, 1024), (1100, 7168, 4096), (1500, 512, 6144), (1100, 512, 8192), (4096, 1536, 5120),
    # tiles of 128 x 128: two and four buffers, k whole and split
    (8192, 4096, 64), (1500, 128, 256), (8192, 14336, 16), (8192, 4096, 256), (512, 14336, 1024), (300, 28672, 512),
    # rings of one block of rows, k whole and split
    (33, 640, 14336), (50, 5120, 5120), (50, 640, 16384), (128, 256, 14336), (33, 512, 28672), (50, 512, 28672),
    (100, 128, 28672),
]


def exact_case(m, k, n, dtype, seed):
    """Operands whose products, scaled, are multiples of 1/4 with sums below 2^21: fp32 holds them all, and the matrix
    unit, which keeps 13 bits below a group's largest product (at most 4, a multiple of 1), drops nothing."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def ints(shape):
        return torch.randint(-1, 3, shape, generator=g, device="cuda").float()

    def scales(shape):
        return torch.exp2(torch.randint(-1, 2, shape, generator=g, device="cuda").float())

    q, w = ints((m, k)).to(E4), ints((n, k)).to(E4)
    s, ws = scales((m, -(-k // 128))), scales((-(-n // 128), -(-k // 128)))
    bias = ints((n,)).to(dtype) if seed & 1 else None
    y = (q.double() * s.double().repeat_interleave(128, 1)[:, :k]) @ weight64(w, ws).t()
    if bias is not None:
        y += bias.double()
    return q, s, w, ws, bias, y.to(dtype)


def call(q, s, w, ws, bias, dtype, buf, nbytes):
    """The product through the C entry, in front of and behind it 64 numbers that stay as they were."""
    m, k, n = *q.shape, w.shape[0]
    y = torch.full((m * n + 128,), 7.0, dtype=dtype, device="cuda")
    rc = _lib.lib().exl3_fp8_linear(q.data_ptr(), _lib.DTYPE_E4M3, s.data_ptr(), w.data_ptr(), ws.data_ptr(),
                                    None if bias is None else bias.data_ptr(), y[64:].data_ptr(),
                                    _lib.DTYPE_BF16 if dtype == BF else _lib.DTYPE_F16, m, k, n,
                                    None if buf is None else buf.data_ptr(), nbytes, stream())
    assert rc == 0, _lib.lib().exl3_last_error()
    assert (y[:64] == 7).all() and (y[64 + m * n:] == 7).all()
    return y[64:64 + m * n].view(m, n)


COUNTERS = 256 * 1024


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_every_kernel_exactly(m, k, n, ragged):
    if ragged:  # columns of k that end inside a block, rows of y that no wide store fits, another type, a bias
        k, n = k - 16, n + 5
    print(f"case: {m} x {k} x {n}", flush=True)
    dtype = HF if ragged else BF
    q, s, w, ws, bias, want = exact_case(m, k, n, dtype, 2 * (m + k) + ragged)
    need = int(_lib.lib().exl3_fp8_linear_workspace_size(_lib.DTYPE_E4M3, m, k, n))
    buf = torch.full((need,), 255, dtype=torch.uint8, device="cuda") if need else None  # scratch: NaNs
    if need:
        buf[:COUNTERS] = 0
    for _ in range(2):
        assert torch.equal(call(q, s, w, ws, bias, dtype, buf, need), want)
        assert not need or not buf[:COUNTERS].any()
    if need:  # k is split: without room for the sums it is not
        assert torch.equal(call(q, s, w, ws, bias, dtype, None, 0), want)
        assert torch.equal(call(q, s, w, ws, bias, dtype, buf, need - 1), want)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,k,n", [(1, 128, 16), (1, 512, 16), (2, 4096, 16), (1, 4096, 6144), (4, 2048, 1536),
                                   (3, 4096, 2048), (4, 16384, 300), (1, 14336, 4096), (24, 2064, 515), (200, 1024, 640)])
def test_rows_quantized_on_the_way_exactly(m, k, n, dtype):
    """16-bit rows whose every group has a 448 and is scaled by 1/2, 1 or 2: they are that scale and whole numbers.
    A product is at most 896, so that a group of 16 keeps multiples of 2^-4; the sums stay below 2^21
    (128 groups' can pass 65504: an infinity in fp16, here as in the rounded 64-bit sum)."""
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    groups = -(-k // 128)
    q = torch.randint(-1, 3, (m, k), generator=g, device="cuda").float()
    at = torch.arange(groups, device="cuda") * 128 + torch.randint(0, 16, (m, groups), generator=g, device="cuda")
    q.scatter_(1, at, 448.0)
    s = torch.exp2(torch.randint(-1, 2, (m, groups), generator=g, device="cuda").float())
    _, _, w, ws, _, _ = exact_case(1, k, n, dtype, 4)
    x64 = q.double() * s.double().repeat_interleave(128, 1)[:, :k]
    want = (x64 @ weight64(w, ws).t()).to(dtype)
    got = op().fp8_linear(x64.to(dtype), w, ws, None, None, dtype == BF)
    assert torch.equal(got, want)
    assert torch.equal(op().fp8_linear(q.to(E4), w, ws, s, None, dtype == BF), want)


@pytest.mark.parametrize("m,k,n", [(1, 1024, 16), (12, 5120, 16), (100, 5120, 1536), (65, 640, 6144), (300, 1024, 4096),
                                   (512, 14336, 256), (1500, 512, 6144)])
def test_fp16_results_keep_small_products(m, k, n):
    """256 - 256 + 2^-9 in a block: 17 bits apart, within fp32's 24 and beyond the 13 that the e4m3 unit keeps."""
    q, w = torch.zeros((m, k), device="cuda"), torch.zeros((n, k), device="cuda")
    for at in ((0, 1, 2), (128, 192, 255), (k - 16, k - 9, k - 1)):
        q[:, at[0]], q[:, at[1]], q[:, at[2]] = 16.0, 16.0, 2.0 ** -9
        w[:, at[0]], w[:, at[1]], w[:, at[2]] = 16.0, -16.0, 1.0
    s, ws = torch.ones((m, -(-k // 128)), device="cuda"), torch.ones((-(-n // 128), -(-k // 128)), device="cuda")
    y = op().fp8_linear(q.to(E4), w.to(E4), ws, s, None, False)
    assert torch.equal(y, torch.full_like(y, 3 * 2.0 ** -9))


@pytest.mark.parametrize("m,k,n", [(1, 272, 200), (4, 272, 200), (40, 5120, 300), (300, 1024, 200), (1500, 272, 6144)])
def test_bad_values_of_fp16_stay_in_their_row(m, k, n):
    x, (w, ws) = make_rows(m, k, 7, HF), make_weight(n, k, 8)
    r = m // 2
    for bad in (float("inf"), float("-inf"), float("nan")):
        x[r, k - 2] = bad
        y = op().fp8_linear(x, w, ws, None, None, False)
        assert y[r].isnan().all() and torch.cat((y[:r], y[r + 1:])).isfinite().all()
    x[r, k - 2] = 1.0
    w.view(torch.uint8)[131, 5] = 0xFF
    y = op().fp8_linear(x, w, ws, None, None, False)
    assert y[:, 131].isnan().all() and torch.cat((y[:, :131], y[:, 132:]), 1).isfinite().all()


def test_a_limit_that_fp32_cannot_hold_is_refused():
    x = make_rows(2, 64, 1)
    for limit in (1e-40, 5e-324):
        with pytest.raises(RuntimeError, match="least normal"):
            op().fp8_swiglu_quant(x, limit)
    q, s = op().fp8_swiglu_quant(x, 2.0 ** -126)
    assert (s == float(torch.tensor(1e-10) / 448)).all() and (q.float() == 0).all()


@pytest.mark.parametrize("off", [1, 4])
@pytest.mark.parametrize("m,k,n", [(1, 256, 64), (40, 256, 192), (300, 512, 1024), (1500, 256, 6144)])
def test_outputs_at_any_address(m, k, n, off):
    """y at 2 and 8 bytes: narrow stores."""
    q, s, w, ws, bias, want = exact_case(m, k, n, BF, 5)
    y = torch.full((m * n + 16,), 7.0, dtype=BF, device="cuda")
    rc = _lib.lib().exl3_fp8_linear(q.data_ptr(), _lib.DTYPE_E4M3, s.data_ptr(), w.data_ptr(), ws.data_ptr(),
                                    bias.data_ptr(), y[off:].data_ptr(), _lib.DTYPE_BF16, m, k, n, None, 0, stream())
    assert rc == 0
    assert torch.equal(y[off:off + m * n].view(m, n), want)
    assert (y[:off] == 7).all() and (y[off + m * n:] == 7).all()


def test_norm_in_place():
    """Packed rows: the sum over the residual or x, the normed rows over x."""
    m, k = 37, 2064
    x, res = make_rows(m, k, 1), make_rows(m, k, 2)
    w = make_rows(1, k, 3)[0]
    want = op().fp8_norm_quant(x, w, 1e-5, res, True)
    for into in ("residual", "x"):
        a, b = x.clone(), res.clone()
        q, s = torch.empty((m, k), dtype=E4, device="cuda"), torch.empty((m, -(-k // 128)), device="cuda")
        rows = torch.empty_like(a) if into == "x" else a
        rc = _lib.lib().exl3_fp8_norm_quant(a.data_ptr(), k, b.data_ptr(), k, w.data_ptr(), 1e-5,
                                            (a if into == "x" else b).data_ptr(), rows.data_ptr(), q.data_ptr(),
                                            s.data_ptr(), _lib.DTYPE_BF16, m, k, stream())
        assert rc == 0
        for got, ref in zip((q, s, a if into == "x" else b, rows), want):
            assert torch.equal(got.float(), ref.float())


@pytest.mark.parametrize("m,k", [(1025, 4096), (1025, 4080), (1024, 4096), (2, 4112), (3, 8192), (3, 8208), (2, 16384)])
def test_norm_rows_of_every_width(m, k):
    """One, two and four chunks a thread, on both sides of where they change."""
    x, res, w = make_rows(m, k, 1, HF), make_rows(m, k, 2, HF), make_rows(1, k, 3, HF)[0]
    q, s, h, rows = op().fp8_norm_quant(x, w, 1e-5, res, True)
    _, y = norm64(x, w, 1e-5, res)
    # the sum of squares: chains of at most 32, a tree of 22 steps; half of it, with the mean's 4, comes out of the
    # root; root, quotient and products are 8 more
    slack = ((32 + 22 + 4) / 2 + 8) * U
    check_quant(q, s, y, slack, f"{m} x {k}")
    assert torch.equal(h, (x.float() + res.float()).half())
    bound = (2.0 ** -11 * 1.001 + slack) * y.abs() + 2.0 ** -24
    assert bool(((rows.double() - y).abs() <= bound).all())


def test_norm_beyond_fp32():
    """A mean square beyond fp32 gives zeros, as documented; its neighbours are not touched by it."""
    x = make_rows(3, 256, 1)
    w = torch.ones(256, dtype=BF, device="cuda")
    want = op().fp8_norm_quant(x, w, 1e-6, None, True)
    x[1] = 3e38
    got = op().fp8_norm_quant(x, w, 1e-6, None, True)
    assert (got[2][1] == 0).all() and (got[0][1].float() == 0).all()
    for r in (0, 2):
        assert torch.equal(got[2][r], want[2][r])
    assert norm64(x, w, 1e-6)[1].isfinite().all()


# ----------------------------------------------------- native and general entries

def _bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def _same(a, b):
    a, b = (list(t) if isinstance(t, (tuple, list)) else [t] for t in (a, b))
    assert len(a) == len(b)
    for s, t in zip(a, b):
        assert s.shape == t.shape and s.dtype == t.dtype and s.stride() == t.stride() and torch.equal(_bits(s), _bits(t))


def _forms(x):
    """x, and the same numbers in other layouts."""
    wide = torch.zeros((x.shape[0], x.shape[1] + 40), dtype=x.dtype, device="cuda")
    wide[:, 8:8 + x.shape[1]] = x
    odd = torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")
    odd[1:] = x.reshape(-1)
    return [x, x.view(2, -1, x.shape[1]), wide[:, 8:8 + x.shape[1]], odd[1:].view(x.shape), x.t().contiguous().t(), x[:1],
            x[0], x[::2], x[:0]]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m", [2, 40, 300])
def test_native_and_general(m, dtype):
    o, k, n = op(), 544, 208
    w, ws = make_weight(n, k, 1)
    gain = make_rows(1, k, 2, dtype)[0]
    bias = make_rows(1, n, 3, dtype)[0]

    def calls():
        for x, res in zip(_forms(make_rows(m, k, 4, dtype)), _forms(make_rows(m, k, 5, dtype))):
            _same(o.fp8_quant_rows(x), o.fp8_quant_rows_general(x))
            _same(o.fp8_swiglu_quant(x, 2.0), o.fp8_swiglu_quant_general(x, 2.0))
            for r, rows in ((None, False), (res, False), (res, True), (None, True)):
                _same(o.fp8_norm_quant(x, gain, 1e-5, r, rows), o.fp8_norm_quant_general(x, gain, 1e-5, r, rows))
            q, s = o.fp8_quant_rows(x)
            for b, out in ((None, True), (bias, dtype == BF)):
                _same(o.fp8_linear(x, w, ws, None, b, out), o.fp8_linear_general(x, w, ws, None, b, out))
                _same(o.fp8_linear(q, w, ws, s, b, out), o.fp8_linear_general(q, w, ws, s, b, out))

    calls()
    with torch.inference_mode():
        calls()
    errors = []

    def other():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                calls()
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001 - handed to the test's thread
            errors.append(e)

    t = threading.Thread(target=other)
    t.start()
    t.join()
    if errors:
        raise errors[0]


def test_inputs_that_require_grad():
    """The operators have no gradient: their outputs do not ask for one that could not be computed."""
    o = op()
    x, (w, ws) = make_rows(4, 256, 1).requires_grad_(), make_weight(64, 256, 2)
    gain = torch.ones(256, dtype=BF, device="cuda", requires_grad=True)
    _same(o.fp8_quant_rows(x)[0].detach(), o.fp8_quant_rows(x.detach())[0])
    _same(o.fp8_norm_quant(x, gain, 1e-6)[0].detach(), o.fp8_norm_quant(x.detach(), gain.detach(), 1e-6)[0])
    y = o.fp8_linear(x, w, ws)
    _same(y.detach(), o.fp8_linear(x.detach(), w, ws))
    if y.requires_grad:
        with pytest.raises(RuntimeError):
            y.float().sum().backward()


# ------------------------------------------------------------ graphs, workspaces

def test_two_graphs_of_one_stream():
    """They share the stream's workspace, and run one after the other on it; the larger call's came first."""
    o = op()
    k = 5120
    sizes = [(17, 4096), (100, 1536), (400, 1536)]
    sets = [(make_rows(m, k, m), *make_weight(n, k, n)) for m, n in sizes]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        want = [o.fp8_linear(*a).clone() for a in sets]
        graphs, outs = [], []
        for a in sets:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                outs.append(o.fp8_linear(*a))
            graphs.append(g)
        for _ in range(3):
            for i in (0, 1, 2, 1, 0):
                outs[i].zero_()
                graphs[i].replay()
                assert torch.equal(o.fp8_linear(*sets[2 - i]), want[2 - i])
                assert torch.equal(outs[i], want[i])
    st.synchronize()
    for (x, w, ws), y in zip(sets, want):
        q, s = o.fp8_quant_rows(x)
        check_product(y, q, s, w, ws)


def test_capture_needs_a_workspace_that_is_there():
    """A stream that never ran such a call has none: the capture is refused, and what follows works."""
    o = op()
    x, (w, ws) = make_rows(40, 1024, 1), make_weight(512, 1024, 2)
    want = o.fp8_linear(x, w, ws)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=st):
            o.fp8_linear(x, w, ws)
    with torch.cuda.stream(st):
        assert torch.equal(o.fp8_linear(x, w, ws), want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            y = o.fp8_linear(x, w, ws)
        for _ in range(3):
            y.zero_()
            g.replay()
            assert torch.equal(y, want)
    torch.cuda.current_stream().wait_stream(st)
