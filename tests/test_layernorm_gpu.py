"""Layer norm, forward and backward, against plain 64-bit formulas.

Tolerances (u = 2^-24, the rounding of one fp32 operation; h the normalised value):
an fp32 sum in the kernels adds at most 64 values after one another plus a tree, so a
mean carries at most D u times the mean magnitude, D = 96 for rows in registers. That
error of the mean, u |x| of the centring and the same again through rstd give
|y - exact| <= D u rstd max|x| (1 + |h|) |gamma| + 4 u (|h gamma| + |beta|), and one
rounding to the result's type. Rows read in pieces add up to cols / 1024 values per
thread: D grows by that.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from tests._gpu import require_gpu, torch  # noqa: E402

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def pk():
    require_gpu()
    import pkt_b200
    return pkt_b200


def ptr(t):
    return None if t is None else t.data_ptr()


def kind(pk, t):
    return {torch.bfloat16: pk.DTYPE_BF16, torch.float32: pk.DTYPE_F32}[t]


def padded(rows, ld, dtype, offset=0, fill=7.0):
    """[rows, ld] that starts `offset` elements into its memory; the guard holds `fill`."""
    flat = torch.full((rows * ld + offset + 64,), fill, dtype=dtype, device="cuda")
    return flat[offset:offset + rows * ld].view(rows, ld), flat


def make(pk, rows, cols, dtype="bf16", params="f32", pad=0, offset=0, affine=True, seed=0, mean=0.5, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, p = TYPES[dtype], TYPES[params]
    x, _ = padded(rows, cols + pad, t, offset)
    dy, _ = padded(rows, cols + pad, t, offset)
    x[:, :cols] = (torch.randn(rows, cols, generator=g, device="cuda") * scale + mean).to(t)
    dy[:, :cols] = torch.randn(rows, cols, generator=g, device="cuda").to(t)
    gamma = (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).to(p) if affine else None
    beta = (0.3 * torch.randn(cols, generator=g, device="cuda")).to(p) if affine else None
    y, yflat = padded(rows, cols + pad, t, offset)
    dx, dxflat = padded(rows, cols + pad, t, offset)
    s = dict(x=x, dy=dy, gamma=gamma, beta=beta, y=y, dx=dx, mean=torch.full((rows,), 9.0, device="cuda"),
             rstd=torch.full((rows,), 9.0, device="cuda"), dgamma=torch.full((cols,), 9.0, device="cuda"),
             dbeta=torch.full((cols,), 9.0, device="cuda"), cols=cols, guards=[(y, yflat, offset), (dx, dxflat, offset)])
    d = pk.LayerNormDesc(rows=rows, cols=cols, dtype=kind(pk, t), param_dtype=kind(pk, p), eps=1e-5,
                         x=ptr(x), ldx=x.stride(0) if rows else cols, gamma=ptr(gamma), beta=ptr(beta), y=ptr(y), ldy=cols + pad,
                         mean=ptr(s["mean"]), rstd=ptr(s["rstd"]), dy=ptr(dy), lddy=cols + pad, dx=ptr(dx), lddx=cols + pad,
                         dgamma=ptr(s["dgamma"]), dbeta=ptr(s["dbeta"]))
    s["work"] = torch.empty(pk.layernorm_backward_workspace(d), dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = ptr(s["work"]), s["work"].numel()
    return d, s


def exact_forward(s, eps=1e-5):
    x = s["x"][:, :s["cols"]].double()
    mean = x.mean(1)
    c = x - mean[:, None]
    rstd = 1 / torch.sqrt((c * c).mean(1) + eps)
    h = c * rstd[:, None]
    g = s["gamma"].double() if s["gamma"] is not None else torch.ones(s["cols"], dtype=torch.float64, device="cuda")
    b = s["beta"].double() if s["beta"] is not None else torch.zeros(s["cols"], dtype=torch.float64, device="cuda")
    return x, mean, rstd, h, g, b


def half(t):
    return torch.finfo(t).eps / 2


def depth(cols):
    return 96 + cols / 1024


def check_forward(s):
    x, mean, rstd, h, g, b = exact_forward(s)
    y = h * g + b
    big = x.abs().amax(1, keepdim=True)
    D = depth(s["cols"])
    tol = D * U * rstd[:, None] * big * (1 + h.abs()) * g.abs() + 4 * U * ((h * g).abs() + b.abs())
    tol = tol + half(s["y"].dtype) * (y.abs() + tol)
    got = s["y"][:, :s["cols"]].double()
    assert torch.all((got - y).abs() <= tol), float(((got - y).abs() / tol).max())
    assert torch.all((s["mean"].double() - mean).abs() <= D * U * big[:, 0])
    assert torch.all((s["rstd"].double() - rstd).abs() <= (2 * D * U * big[:, 0] * rstd + (D + 4) * U) * rstd)


def check_guards(s, which):
    for t, flat, offset in s["guards"]:
        if t is not s[which]:
            continue
        assert torch.all(t[:, s["cols"]:] == 7.0)
        assert torch.all(flat[:offset] == 7.0) and torch.all(flat[offset + t.numel():] == 7.0)


def check_backward(s, want_dx=True):
    """From the kernel's own mean and rstd, which are inputs of the backward pass."""
    cols = s["cols"]
    x, dy = s["x"][:, :cols].double(), s["dy"][:, :cols].double()
    mean, rstd = s["mean"].double()[:, None], s["rstd"].double()[:, None]
    g = s["gamma"].double() if s["gamma"] is not None else torch.ones(cols, dtype=torch.float64, device="cuda")
    h, w = (x - mean) * rstd, dy * g
    c1, c2 = w.mean(1, keepdim=True), (w * h).mean(1, keepdim=True)
    dx = rstd * (w - c1 - h * c2)
    # the row sums: D u of their mean magnitude; h: 2 u; then 6 operations
    D = depth(cols)
    m1, m2 = w.abs().mean(1, keepdim=True), (w * h).abs().mean(1, keepdim=True)
    tol = rstd * (D * U * (m1 + h.abs() * m2) + 8 * U * (w.abs() + c1.abs() + (h * c2).abs() + h.abs() * m2))
    tol = tol + half(s["dx"].dtype) * (dx.abs() + tol)
    if want_dx:
        got = s["dx"][:, :cols].double()
        assert torch.all((got - dx).abs() <= tol), float(((got - dx).abs() / tol).max())
    # the column sums: a thread adds rows / 296 values at most (2 blocks per SM), the rest is a tree of 64
    D = 64 + x.shape[0] / 296 + 4
    tol = D * U * (dy * h).abs().sum(0)
    assert torch.all((s["dgamma"].double() - (dy * h).sum(0)).abs() <= tol)
    assert torch.all((s["dbeta"].double() - dy.sum(0)).abs() <= D * U * dy.abs().sum(0))


SHAPES = [(1, 1), (2, 2), (3, 7), (1, 64), (5, 100), (17, 128), (33, 256), (300, 512), (700, 777), (1200, 96), (64, 1024), (601, 1024),
          (40, 4096), (700, 4096), (9, 4097), (310, 5000), (3, 8192), (320, 8192), (4, 8200), (2, 16384), (5, 20001), (2, 40000)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_backward(pk, rows, cols, dtype):
    d, s = make(pk, rows, cols, dtype, params="f32" if cols % 2 else "bf16", seed=rows + cols)
    pk.layernorm_forward(d)
    check_forward(s)
    check_guards(s, "y")
    pk.layernorm_backward(d)
    check_backward(s)
    check_guards(s, "dx")


@pytest.mark.parametrize("pad,offset", [(8, 0), (1, 0), (0, 1), (24, 8), (3, 5)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(37, 333), (700, 640), (5, 9000)])
def test_strides_and_alignment(pk, rows, cols, dtype, pad, offset):
    d, s = make(pk, rows, cols, dtype, pad=pad, offset=offset, seed=pad + offset)
    pk.layernorm_forward(d)
    check_forward(s)
    check_guards(s, "y")
    pk.layernorm_backward(d)
    check_backward(s)
    check_guards(s, "dx")


def test_no_affine_no_statistics(pk):
    d, s = make(pk, 50, 300, affine=False)
    pk.layernorm_forward(d)
    check_forward(s)
    pk.layernorm_backward(d)
    check_backward(s)
    first = s["y"].clone()
    d.mean = d.rstd = None
    s["y"].zero_()
    pk.layernorm_forward(d)
    assert torch.equal(s["y"], first)


def test_only_weight_gradients_and_only_dx(pk):
    d, s = make(pk, 400, 520)
    pk.layernorm_forward(d)
    d.dx = None
    pk.layernorm_backward(d)
    check_backward(s, want_dx=False)
    assert torch.all(s["dx"] == 7.0)
    d.dx, d.dgamma, d.dbeta = ptr(s["dx"]), None, None
    keep = s["dgamma"].clone()
    pk.layernorm_backward(d)
    check_backward(s)
    assert torch.equal(s["dgamma"], keep)


def test_large_mean_small_spread(pk):
    """The variance is taken of the centred values: a mean of 1000 spreads does not eat it."""
    d, s = make(pk, 64, 1024, "f32", mean=1000.0)
    pk.layernorm_forward(d)
    check_forward(s)


def test_constant_and_nonfinite_rows(pk):
    d, s = make(pk, 6, 200, "f32")
    s["x"][0] = 3.0          # no spread: rstd is 1/sqrt(eps), y is beta
    s["x"][2, 5] = float("inf")
    s["x"][4, 199] = float("nan")
    pk.layernorm_forward(d)
    y = s["y"]
    assert torch.equal(y[0], s["beta"])
    assert torch.all(torch.isnan(y[2])) and torch.all(torch.isnan(y[4]))
    assert torch.all(torch.isfinite(y[[1, 3, 5]]))  # the rows beside them are untouched


def test_in_place(pk):
    for cols in (300, 9000):
        d, s = make(pk, 30, cols)
        pk.layernorm_forward(d)
        want = s["y"].clone()
        pk.layernorm_backward(d)
        dx = s["dx"].clone()
        d.dx = d.dy
        pk.layernorm_backward(d)
        assert torch.equal(s["dy"], dx)
        d.y = d.x
        pk.layernorm_forward(d)
        assert torch.equal(s["x"], want)


def test_no_rows(pk):
    d, s = make(pk, 1, 100)
    d.rows = 0
    d.x = d.y = d.dy = d.dx = d.mean = d.rstd = d.workspace = None
    pk.layernorm_forward(d)
    pk.layernorm_backward(d)
    assert torch.all(s["dgamma"] == 0) and torch.all(s["dbeta"] == 0) and torch.all(s["y"] == 7.0)


def test_repeats_are_identical(pk):
    d, s = make(pk, 5000, 260)
    pk.layernorm_forward(d)
    pk.layernorm_backward(d)
    a, b = s["dgamma"].clone(), s["dbeta"].clone()
    for _ in range(5):
        pk.layernorm_backward(d)
        assert torch.equal(s["dgamma"], a) and torch.equal(s["dbeta"], b)


def test_offsets_past_32_bits(pk):
    """A row stride of more than 2^30 elements: the third row starts past 2^32 bytes."""
    rows, cols, ld = 3, 264, (1 << 30) + 8
    d, s = make(pk, rows, cols)
    big = torch.empty((rows - 1) * ld + cols, dtype=torch.bfloat16, device="cuda")
    view = torch.as_strided(big, (rows, cols), (ld, 1))
    view.copy_(s["x"])
    d.x, d.ldx = ptr(big), ld
    pk.layernorm_forward(d)
    check_forward(s)
    pk.layernorm_backward(d)
    check_backward(s)
    d.x, d.ldx, d.y, d.ldy = ptr(s["x"]), cols, ptr(big), ld
    pk.layernorm_forward(d)
    assert torch.equal(view, s["y"])


def test_streams_and_graph(pk):
    d, s = make(pk, 900, 1000)
    pk.layernorm_forward(d)
    pk.layernorm_backward(d)
    want = {k: s[k].clone() for k in ("y", "dx", "dgamma", "dbeta")}
    st = torch.cuda.Stream()
    for k in want:
        s[k].fill_(1.0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        pk.layernorm_forward(d, st.cuda_stream)
        pk.layernorm_backward(d, st.cuda_stream)
    assert torch.all(s["y"] == 1.0)  # captured, not run
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for k, v in want.items():
        assert torch.equal(s[k], v), k
    # a new input through the same graph
    s["x"].mul_(-1)
    g.replay()
    torch.cuda.synchronize()
    check_forward(s)
    check_backward(s)


def test_gradients_against_differences(pk):
    """dx, dgamma, dbeta of L = sum(dy * y) against central differences of the fp64 formula."""
    d, s = make(pk, 3, 40, "f32", seed=4)
    pk.layernorm_forward(d)
    pk.layernorm_backward(d)
    x, g, b, dy = (s[k].double() for k in ("x", "gamma", "beta", "dy"))

    def loss(x, g, b):
        c = x - x.mean(1, keepdim=True)
        return float((dy * (c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * g + b)).sum())

    e = 1e-5
    for k, t, got in ((0, x, s["dx"]), (1, g, s["dgamma"]), (2, b, s["dbeta"])):
        args = [x, g, b]
        for i in np.random.default_rng(0).choice(t.numel(), 20, replace=False):
            up, down = t.clone().view(-1), t.clone().view(-1)
            up[i] += e
            down[i] -= e
            args[k] = up.view(t.shape)
            hi = loss(*args)
            args[k] = down.view(t.shape)
            diff = (hi - loss(*args)) / (2 * e)
            # truncation e^2 and rounding 2^-53 |L| / e are below 1e-8; the fp32 result carries ~100 u
            assert abs(float(got.reshape(-1)[i]) - diff) <= 1e-5 * (1 + abs(diff))


def test_refuses_what_it_cannot_reach(pk):
    d, s = make(pk, 8, 64)
    host = torch.zeros(8, 64, dtype=torch.bfloat16)
    d.x = host.data_ptr()
    with pytest.raises(pk.PktError, match="x is not device memory"):
        pk.layernorm_forward(d)
    d.x = ptr(s["x"])
    d.workspace_bytes -= 1
    with pytest.raises(pk.PktError, match="workspace of"):
        pk.layernorm_backward(d)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(40000, 4), (20000, 8), (9001, 64), (5000, 96), (12000, 128), (30000, 7)])
def test_many_short_rows(pk, rows, cols, dtype):
    d, s = make(pk, rows, cols, dtype, seed=cols)
    pk.layernorm_forward(d)
    check_forward(s)
    pk.layernorm_backward(d)
    check_backward(s)


@pytest.mark.parametrize("dtype,pad", [("bf16", 0), ("bf16", 1), ("f32", 0)])
def test_rows_of_many_millions(pk, dtype, pad):
    """More slabs of columns than one grid dimension but the first can count."""
    d, s = make(pk, 2, 65536 * 512 + 1032, dtype, pad=pad, seed=pad)
    pk.layernorm_forward(d)
    check_forward(s)
    pk.layernorm_backward(d)
    check_backward(s)


def test_in_place_through_the_rings(pk):
    """Rows that share 16-byte granules with their neighbours, read ahead while earlier ones are written."""
    for cols, dtype in ((777, "bf16"), (1024, "bf16"), (333, "f32")):
        d, s = make(pk, 6000, cols, dtype)
        pk.layernorm_forward(d)
        want = s["y"].clone()
        pk.layernorm_backward(d)
        dx = s["dx"].clone()
        for into in ("dy", "x"):
            keep = s[into].clone()
            d.dx = ptr(s[into])
            pk.layernorm_backward(d)
            assert torch.equal(s[into], dx)
            s[into].copy_(keep)
        d.y = d.x
        pk.layernorm_forward(d)
        assert torch.equal(s["x"], want)


def test_two_calls_at_once(pk):
    """Two streams, a workspace each."""
    a, b = make(pk, 3000, 1000, seed=1), make(pk, 2500, 777, "f32", seed=2)
    for d, s in (a, b):
        pk.layernorm_forward(d)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        for (d, s), st in zip((a, b), streams):
            pk.layernorm_backward(d, st.cuda_stream)
            pk.layernorm_forward(d, st.cuda_stream)
    torch.cuda.synchronize()
    for d, s in (a, b):
        check_forward(s)
        check_backward(s)


@pytest.mark.parametrize("dtype,pad", [("f32", 0), ("f32", 1), ("bf16", 0), ("bf16", 1)])
@pytest.mark.parametrize("rows,cols", [(6, 1000), (6, 777), (3000, 1000), (3000, 777), (5000, 40), (5000, 41), (700, 6000), (700, 6007), (3, 20000), (3, 24999), (3, 25001)])
def test_rows_without_spread(pk, rows, cols, dtype, pad):
    """Every partial sum of these values is exact in any order, so the mean is the value and y is beta
    (directly loaded rows, rows through the rings, long rows; whole and one by one)."""
    d, s = make(pk, rows, cols, dtype, pad=pad, seed=cols)
    values = [3.0, 100.0, -7.0, 0.75, 113.0, 1.0]
    for i, v in enumerate(values):
        s["x"][i::len(values), :cols] = v
    pk.layernorm_forward(d)
    assert torch.equal(s["mean"], s["x"][:, 0].float())
    assert torch.equal(s["y"][:, :cols], s["beta"].to(TYPES[dtype]).expand(rows, cols))
    check_guards(s, "y")
