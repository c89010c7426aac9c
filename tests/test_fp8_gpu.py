"""Block-scaled 8-bit floats: the quantiser against its definition (bit for bit and in
64 bits), the product against the 64-bit sum of the values its operands stand for.

Tolerances. Quantiser: scale = amax / most is one rounding (2^-24); q stands for
x * (most / amax), two roundings, then half a step of the type: |q s - x| <=
(half + 4 2^-24) |x| + s smallest / 2. Product: the tensor core adds 32 products at a
time to an fp32 accumulator, the blocks of 128 are scaled and added in fp32. With
every partial sum off by at most 2^-22 of the sum of magnitudes per addition (fp32
accumulation that may truncate), 4 additions per block and one per block of K,
|out - exact| <= (4 + blocks) 2^-22 sum |terms| + one rounding to the result's type.
"""
import pytest

pytestmark = pytest.mark.gpu

from tests._gpu import require_gpu, torch  # noqa: E402

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TINY = 2.0 ** -100


@pytest.fixture(scope="module")
def pk():
    require_gpu()
    import pkt_b200
    return pkt_b200


def kind(pk, name):
    return {"bf16": pk.DTYPE_BF16, "f32": pk.DTYPE_F32, "e4m3": pk.DTYPE_E4M3, "e5m2": pk.DTYPE_E5M2}[name]


def up(n, k=16):
    return -(-n // k) * k


# ---------------------------------------------------------------- quantiser
def quantise(pk, x, q="e4m3", block_rows=1, plain=True, transposed=False, cols=None, stream=None):
    """Runs the quantiser into guarded outputs; returns {q, scale, qt, scale_t} without the guards."""
    rows, cols = x.shape[0], cols or x.shape[1]
    t = TYPES[q]
    out, guards = {}, []

    def room(n, m, ld):
        flat = torch.full((n * ld + 64,), 3.0, device="cuda").to(t)
        guards.append((flat, n, m, ld))
        return flat[:n * ld].view(n, ld)

    d = pk.Fp8QuantizeDesc(rows=rows, cols=cols, dtype=kind(pk, "bf16" if x.dtype == torch.bfloat16 else "f32"), q_dtype=kind(pk, q),
                           block_rows=block_rows, x=x.data_ptr(), ldx=x.stride(0))
    if plain:
        w = room(rows, cols, up(cols) + 16)
        s = torch.full((-(-cols // 128), -(-rows // block_rows) + 3), 9.0, device="cuda")
        d.q, d.ldq, d.scale, d.ld_scale = w.data_ptr(), w.stride(0), s.data_ptr(), s.stride(0)
        out |= {"q": w[:, :cols], "scale": s}
    if transposed:
        w = room(cols, rows, up(rows) + 16)
        s = torch.full((-(-rows // 128), -(-cols // block_rows) + 3), 9.0, device="cuda")
        d.qt, d.ldqt, d.scale_t, d.ld_scale_t = w.data_ptr(), w.stride(0), s.data_ptr(), s.stride(0)
        out |= {"qt": w[:, :rows], "scale_t": s}
    pk.fp8_quantize(d, stream)
    torch.cuda.synchronize()
    for flat, n, m, ld in guards:
        f = flat.float()
        assert torch.all(f[:n * ld].view(n, ld)[:, m:] == 3.0) and torch.all(f[n * ld:] == 3.0)
    for k in ("scale", "scale_t"):
        if k in out:
            assert torch.all(out[k][:, -3:] == 9.0)
            out[k] = out[k][:, :-3].contiguous()
    return out


def plain_blocks(x, dtype, block_rows):
    """The definition in fp32: [rows, cols] -> q, scale [column blocks, row blocks]."""
    rows, cols = x.shape
    pad = torch.zeros(up(rows, block_rows), up(cols, 128), device="cuda")
    pad[:rows, :cols] = x.float()
    b = pad.view(-1, block_rows, pad.shape[1] // 128, 128)
    big = b.abs().amax((1, 3), keepdim=True)
    most = torch.full_like(big, torch.finfo(dtype).max)
    none = big < TINY
    f, s = torch.where(none, 0.0, most / big), torch.where(none, 0.0, big / most)
    q = (b * f).to(dtype)
    return q.view(pad.shape)[:rows, :cols], s[:, 0, :, 0].t().contiguous()


def values(rows, cols, dtype, seed=0, pad=0, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    flat = torch.zeros(rows * (cols + pad) + offset, device="cuda")
    x = flat[offset:].view(rows, cols + pad)
    x.copy_(torch.randn(rows, cols + pad, generator=g, device="cuda") * torch.exp(2 * torch.randn(rows, 1, generator=g, device="cuda")))
    flat = flat.to(TYPES[dtype])
    return flat[offset:].view(rows, cols + pad)[:, :cols]


SHAPES = [(1, 1), (1, 128), (1, 129), (3, 16), (5, 1000), (127, 128), (128, 128), (129, 257), (300, 640), (1000, 777), (4099, 10)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q", ["e4m3", "e5m2"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantise(pk, rows, cols, block_rows, q, dtype):
    x = values(rows, cols, dtype, seed=rows + cols)
    t = TYPES[q]
    half, least = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps
    for plain, transposed in ((True, False), (True, True), (False, True)):
        got = quantise(pk, x, q, block_rows, plain, transposed)
        for y, name, sname in ((x, "q", "scale"), (x.t(), "qt", "scale_t")):
            if name not in got:
                continue
            wq, ws = plain_blocks(y, t, block_rows)
            assert torch.equal(got[sname], ws), name
            assert torch.equal(got[name].float(), wq.float()), name
            s = ws.double().t().repeat_interleave(block_rows, 0)[:y.shape[0]].repeat_interleave(128, 1)[:, :y.shape[1]]
            err = (got[name].double() * s - y.double()).abs()
            assert torch.all(err <= (half + 2.0 ** -22) * y.double().abs() + s * least * 0.5001), name


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pad,offset", [(1, 0), (4, 0), (0, 1), (7, 3)])
def test_quantise_strides(pk, dtype, pad, offset):
    x = values(200, 333, dtype, pad=pad, offset=offset)
    for block_rows in (1, 128):
        got = quantise(pk, x, "e4m3", block_rows, True, True)
        assert torch.equal(got["q"].float(), plain_blocks(x, TYPES["e4m3"], block_rows)[0].float())
        assert torch.equal(got["qt"].float(), plain_blocks(x.t(), TYPES["e4m3"], block_rows)[0].float())
    got = quantise(pk, x, "e4m3", 1)
    assert torch.equal(got["q"].float(), plain_blocks(x, TYPES["e4m3"], 1)[0].float())


def test_quantise_special_values(pk):
    """Zero and tiny blocks are zeros with scale 0; infinities and NaN show in their block's scale only."""
    x = values(130, 512, "f32", seed=1).contiguous()
    x[0, :128] = 0
    x[1, 128:256] = 2.0 ** -101
    x[2, 300] = float("inf")
    x[3, 400] = float("nan")
    x[4, 0] = -3e38
    for transposed in (False, True):
        got = quantise(pk, x, "e4m3", 1, True, transposed)
        s, q = got["scale"], got["q"].float()
        assert float(s[0, 0]) == 0 and torch.all(q[0, :128] == 0)
        assert float(s[1, 1]) == 0 and torch.all(q[1, 128:256] == 0)
        assert float(s[2, 2]) == float("inf") and torch.isnan(s[3, 3])
        finite = torch.isfinite(s)
        finite[2, 2] = finite[3, 3] = True
        assert torch.all(finite)
        assert torch.isfinite(q[4, :128]).all() and float(q[4, 0]) == -448
    got = quantise(pk, x, "e4m3", 1, False, True)
    bad = ~torch.isfinite(got["scale_t"])
    assert bad.nonzero().tolist() == [[0, 300], [0, 400]]


def test_quantise_offsets_past_32_bits(pk):
    rows, cols, ld = 3, 144, (1 << 30) + 16
    x = values(rows, cols, "bf16")
    big = torch.empty((rows - 1) * ld + cols, dtype=torch.bfloat16, device="cuda")
    view = torch.as_strided(big, (rows, cols), (ld, 1))
    view.copy_(x)
    for transposed in (False, True):
        got = quantise(pk, view, "e4m3", 1, True, transposed)
        assert torch.equal(got["q"].float(), plain_blocks(x, TYPES["e4m3"], 1)[0].float())
    out = torch.zeros(2 * (1 << 31) + cols, dtype=torch.uint8, device="cuda")
    s = torch.zeros(2, 3, device="cuda")
    pk.fp8_quantize(pk.Fp8QuantizeDesc(rows=rows, cols=cols, dtype=pk.DTYPE_BF16, q_dtype=pk.DTYPE_E4M3, block_rows=1, x=x.data_ptr(), ldx=x.stride(0),
                                       q=out.data_ptr(), ldq=1 << 31, scale=s.data_ptr(), ld_scale=3))
    got = torch.as_strided(out, (rows, cols), (1 << 31, 1)).contiguous().view(torch.float8_e4m3fn)
    assert torch.equal(got.float(), plain_blocks(x, TYPES["e4m3"], 1)[0].float())


# ---------------------------------------------------------------- product
def operand(rows, k, name, block_rows, seed, ints=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = up(k) + 16 * (seed % 2)
    x = torch.randn(rows, ld, generator=g, device="cuda") * 40  # the padding holds values too: it must not be read
    s = torch.exp(torch.randn(-(-k // 128), -(-rows // block_rows) + seed % 3, generator=g, device="cuda"))
    if ints:
        x = torch.randint(-8, 9, (rows, ld), generator=g, device="cuda").float()
        s = 2.0 ** torch.randint(-2, 3, s.shape, generator=g, device="cuda").float()
    return x.to(TYPES[name]), s


def product(pk, M, N, K, a="e4m3", b="e4m3", ab=1, bb=128, out="bf16", seed=0, pad=0, ints=False, run=None):
    A, sa = operand(M, K, a, ab, seed, ints)
    B, sb = operand(N, K, b, bb, seed + 1, ints)
    ldo = N + pad
    flat = torch.full((M * ldo + 64,), 5.0, dtype=TYPES[out], device="cuda")
    C = flat[:M * ldo].view(M, ldo)
    d = pk.Fp8GemmDesc(M=M, N=N, K=K, a_dtype=kind(pk, a), b_dtype=kind(pk, b), a=A.data_ptr(), lda=A.stride(0), scale_a=sa.data_ptr(),
                       ld_scale_a=sa.stride(0), a_block_rows=ab, b=B.data_ptr(), ldb=B.stride(0), scale_b=sb.data_ptr(), ld_scale_b=sb.stride(0),
                       b_block_rows=bb, out=C.data_ptr(), ldo=ldo, out_dtype=kind(pk, out))
    (run or pk.fp8_gemm)(d)
    torch.cuda.synchronize()
    assert pk.ops_status() == 0
    assert torch.all(C[:, N:] == 5.0) and torch.all(flat[M * ldo:] == 5.0)
    vals = []
    for x, s, rows, blk in ((A, sa, M, ab), (B, sb, N, bb)):
        vals.append(x[:, :K].double() * s.double().t().repeat_interleave(blk, 0)[:rows].repeat_interleave(128, 1)[:, :K])
    want, mag = vals[0] @ vals[1].t(), vals[0].abs() @ vals[1].abs().t()
    return C[:, :N].double(), want, mag, (A, B, sa, sb, flat, d)


def close(got, want, mag, K, out):
    tol = (4 + -(-K // 128)) * 2.0 ** -22 * mag
    tol = tol + torch.finfo(TYPES[out]).eps / 2 * (want.abs() + tol)
    bad = (got - want).abs() > tol
    assert not torch.any(bad), (int(bad.sum()), float(((got - want).abs() / tol).max()), bad.nonzero()[:4].tolist())


GEMMS = [(1, 16, 32), (1, 1, 1), (8, 4096, 512), (16, 1000, 4096), (17, 256, 640), (33, 300, 1000), (64, 512, 2048), (65, 128, 128),
         (100, 777, 300), (128, 128, 4099), (200, 2000, 1536), (300, 10, 777), (1000, 1000, 128), (1024, 2304, 1024), (2500, 1300, 650),
         (4099, 777, 1000)]


@pytest.mark.parametrize("bb", [1, 128])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", GEMMS)
def test_product(pk, M, N, K, out, bb):
    got, want, mag, _ = product(pk, M, N, K, out=out, bb=bb, seed=M + N + K, pad=(M + N) % 3)
    close(got, want, mag, K, out)


@pytest.mark.parametrize("M,N,K", [(5, 200, 600), (40, 130, 256), (150, 260, 384), (2100, 1100, 512)])
@pytest.mark.parametrize("a,b", [("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")])
def test_product_types(pk, M, N, K, a, b):
    got, want, mag, _ = product(pk, M, N, K, a=a, b=b, out="f32")
    close(got, want, mag, K, "f32")


@pytest.mark.parametrize("M,N,K", [(6, 400, 512), (60, 130, 256), (200, 260, 384), (2100, 1100, 512)])
@pytest.mark.parametrize("ab,bb", [(128, 128), (128, 1)])
def test_product_block_rows(pk, M, N, K, ab, bb):
    got, want, mag, _ = product(pk, M, N, K, ab=ab, bb=bb, out="f32")
    close(got, want, mag, K, "f32")


@pytest.mark.parametrize("M,N,K", [(3, 500, 2048), (64, 300, 200), (130, 129, 130), (2300, 1111, 900)])
def test_product_of_small_integers_is_exact(pk, M, N, K):
    """Small integers and powers of two: every partial sum is exact, so is the result."""
    got, want, _, _ = product(pk, M, N, K, ints=True, out="f32", bb=1)
    assert torch.equal(got, want)


def test_product_zero_length(pk):
    _, _, _, (A, B, sa, sb, flat, d) = product(pk, 8, 32, 64)
    d.K = 0
    pk.fp8_gemm(d)
    assert torch.all(flat[:256] == 0) and torch.all(flat[256:] == 5.0)


def test_product_nan_and_zero_scales(pk):
    """A NaN scale reaches its row only; blocks of scale 0 add nothing."""
    _, _, _, (A, B, sa, sb, flat, d) = product(pk, 200, 256, 512, out="f32")
    sa[:, 7] = 0
    sa[1, 9] = float("nan")
    pk.fp8_gemm(d)
    torch.cuda.synchronize()
    C = flat[:200 * 256].view(200, 256)
    assert torch.all(C[7] == 0) and torch.all(torch.isnan(C[9]))
    rest = [i for i in range(200) if i != 9]
    assert torch.all(torch.isfinite(C[rest]))


def test_product_offsets_past_32_bits(pk):
    M, N, K, ld = 3, 40, 200, 1 << 31
    _, want, mag, (A, B, sa, sb, flat, d) = product(pk, M, N, K, out="f32")
    big = torch.empty((M - 1) * ld + up(K), dtype=torch.uint8, device="cuda")
    torch.as_strided(big, (M, K), (ld, 1)).copy_(A.view(torch.uint8)[:, :K])
    res = torch.zeros(2 * (1 << 30) + N, device="cuda")
    d.a, d.lda, d.out, d.ldo = big.data_ptr(), ld, res.data_ptr(), 1 << 30
    pk.fp8_gemm(d)
    torch.cuda.synchronize()
    close(torch.as_strided(res, (M, N), (1 << 30, 1)).double(), want, mag, K, "f32")


def test_product_streams_and_graph(pk):
    st = torch.cuda.Stream()
    cases = []
    for M, N, K in ((8, 1024, 2048), (100, 300, 500), (2048, 2048, 512)):
        got, want, mag, keep = product(pk, M, N, K)
        cases.append((got.clone(), keep))
    for got, (_, _, _, _, flat, d) in cases:
        flat.fill_(0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        for _, keep in cases:
            pk.fp8_gemm(keep[-1], st.cuda_stream)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    for got, (_, _, _, _, flat, d) in cases:
        assert torch.equal(flat[:d.M * d.N].view(d.M, d.N).double(), got)
    # the same product on two streams at once, into two outputs
    got, (A, B, sa, sb, flat, d) = cases[2]
    other, st2 = torch.zeros_like(flat), torch.cuda.Stream()
    d2 = pk.Fp8GemmDesc.from_buffer_copy(d)
    d2.out = other.data_ptr()
    torch.cuda.synchronize()
    for _ in range(4):
        pk.fp8_gemm(d, st.cuda_stream)
        pk.fp8_gemm(d2, st2.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(flat[:d.M * d.N], other[:d.M * d.N])


def test_refuses_what_it_cannot_reach(pk):
    _, _, _, (A, B, sa, sb, flat, d) = product(pk, 8, 32, 64)
    host = torch.zeros(8, 64, dtype=torch.uint8).pin_memory()
    for field in ("a", "b", "scale_a", "scale_b", "out"):
        bad = pk.Fp8GemmDesc.from_buffer_copy(d)
        setattr(bad, field, host.data_ptr())
        with pytest.raises(pk.PktError, match=f"{field} is not device memory"):
            pk.fp8_gemm(bad)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (130, 5), (300, 131), (700, 778), (20000, 643)])
def test_quantise_between_nans(pk, rows, cols, dtype, block_rows):
    """Rows that start anywhere, in memory that holds NaN elsewhere: the bytes and scales of a contiguous copy."""
    x = torch.randn(rows, cols, generator=torch.Generator(device="cuda").manual_seed(cols), device="cuda").to(TYPES[dtype])

    def run(t):
        q = torch.zeros(rows, up(cols), dtype=torch.uint8, device="cuda")
        s = torch.zeros(-(-cols // 128), -(-rows // block_rows), device="cuda")
        qt = torch.zeros(cols, up(rows), dtype=torch.uint8, device="cuda")
        st = torch.zeros(-(-rows // 128), -(-cols // block_rows), device="cuda")
        out = []
        for both in (False, True):  # rows alone, then both ways
            d = pk.Fp8QuantizeDesc(rows=rows, cols=cols, dtype=kind(pk, dtype), q_dtype=pk.DTYPE_E4M3, block_rows=block_rows, x=t.data_ptr(),
                                   ldx=t.stride(0), q=q.data_ptr(), ldq=q.stride(0), scale=s.data_ptr(), ld_scale=s.stride(0))
            if both:
                d.qt, d.ldqt, d.scale_t, d.ld_scale_t = qt.data_ptr(), qt.stride(0), st.data_ptr(), st.stride(0)
            pk.fp8_quantize(d)
            out += [q.clone(), s.clone(), qt.clone(), st.clone()]
        return out

    aligned = torch.zeros(rows, -(-cols // 8) * 8, dtype=x.dtype, device="cuda")[:, :cols]
    aligned.copy_(x)
    want = run(aligned)
    assert all(torch.all(torch.isfinite(t)) for t in want if t.dtype == torch.float32)
    for offset, pad in ((0, 1), (1, 0), (2, 3), (3, 2), (5, 4)):
        flat = torch.full((rows * (cols + pad) + offset + 8,), float("nan"), dtype=x.dtype, device="cuda")
        t = flat[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
        t.copy_(x)
        for a, b in zip(run(t), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("bb", [1, 128])
@pytest.mark.parametrize("M,N,K,out,pad", [(100, 11, 103, "f32", 1), (658, 9, 103, "f32", 3), (658, 11, 1000, "f32", 5), (3799, 1, 29, "f32", 3),
                                           (300, 65, 128, "bf16", 7), (4261, 222, 103, "bf16", 2), (4261, 223, 300, "bf16", 9),
                                           (4261, 777, 1000, "bf16", 7), (2100, 1111, 600, "f32", 1), (2100, 1100, 600, "bf16", 4),
                                           (40, 11, 200, "f32", 1)])
def test_product_beside_other_columns(pk, M, N, K, out, pad, bb):
    """Rows of out on 16-byte boundaries that end inside 16 bytes: the columns behind them keep their values (`product` looks)."""
    got, want, mag, _ = product(pk, M, N, K, out=out, bb=bb, seed=N, pad=pad)
    close(got, want, mag, K, out)
