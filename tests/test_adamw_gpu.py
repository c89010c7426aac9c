"""AdamW over many tensors, states in 32 and in 8 bits, against 64-bit formulas.

Tolerances (u = 2^-24): m and v are two roundings of each term and the rounding of the
fp32 constants: 4 u (|beta m| + |(1 - beta) g|). The parameter: 3 u |p| plus 16 u of
the step's magnitude (9 operations, two rounded constants). An 8-bit state x = q s is
off by half a step of e4m3: 2^-4 |x|, or s 2^-10 below the normal range, and sqrt(v)
by a whole smallest value (s 2^-9) where it is kept above zero.
"""
import pytest

pytestmark = pytest.mark.gpu

from tests._gpu import require_gpu, torch  # noqa: E402

U = 2.0 ** -24
B1, B2, EPS = 0.9, 0.999, 1e-8
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def pk():
    require_gpu()
    import pkt_b200
    return pkt_b200


class Case:
    """Tensors carved out of one memory per array, each `offset` values off its boundary."""

    def __init__(self, pk, sizes, param="f32", grad="f32", state="f32", copy=True, offset=0, seed=0, decay=0.1, step=0, fresh=False, **kw):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.pk, self.sizes, self.eight = pk, sizes, state == "e4m3"
        room = [-(-n // 128) * 128 + 128 + offset for n in sizes]
        self.at = [sum(room[:i]) + offset for i in range(len(sizes))]
        total = sum(room)

        def rnd(scale, dtype=torch.float32):
            return (torch.randn(total, generator=g, device="cuda") * scale).to(dtype)

        self.p, self.g = rnd(0.1, TYPES[param]), rnd(1e-2, TYPES[grad])
        self.copy = torch.full((total,), 7.0, dtype=torch.bfloat16, device="cuda") if copy else None
        self.scales_at = [sum(-(-n // 128) + 1 for n in sizes[:i]) for i in range(len(sizes))]
        ns = sum(-(-n // 128) + 1 for n in sizes)
        if self.eight:
            self.m = torch.randn(total, generator=g, device="cuda").mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn)
            self.v = torch.randn(total, generator=g, device="cuda").abs_().mul_(100).clamp_(0, 448).to(torch.float8_e4m3fn)
            self.ms = torch.rand(ns, generator=g, device="cuda") * 1e-5
            self.vs = torch.rand(ns, generator=g, device="cuda") * 1e-4 + 1e-6
        else:
            self.m, self.v, self.ms, self.vs = rnd(1e-3), rnd(1e-3) ** 2, None, None
        if fresh:
            for t in (self.m, self.v, self.ms, self.vs):
                if t is not None:
                    t.zero_()
        self.decay = [decay * (i % 2) for i in range(len(sizes))]
        rec = []
        for i, n in enumerate(sizes):
            t = pk.AdamWTensor(param=self.p[self.at[i]:].data_ptr(), grad=self.g[self.at[i]:].data_ptr(), m=self.m[self.at[i]:].data_ptr(),
                               v=self.v[self.at[i]:].data_ptr(), n=n, weight_decay=self.decay[i])
            if self.eight:
                t.m_scale, t.v_scale = self.ms[self.scales_at[i]:].data_ptr(), self.vs[self.scales_at[i]:].data_ptr()
            if copy:
                t.copy_bf16 = self.copy[self.at[i]:].data_ptr()
            rec.append(t)
        self.plan = pk.AdamW(rec, beta1=B1, beta2=B2, eps=EPS, param_dtype=param, grad_dtype=grad, state_dtype=state, step=step, **kw)

    def part(self, t, i):
        return t[self.at[i]:self.at[i] + self.sizes[i]]

    def scale(self, t, i):
        n = self.sizes[i]
        s = t[self.scales_at[i]:self.scales_at[i] + -(-n // 128)]
        return s.double().repeat_interleave(128)[:n]

    def state(self, i):
        if self.eight:
            m = self.part(self.m, i).double() * self.scale(self.ms, i)
            return m, (self.part(self.v, i).double() * self.scale(self.vs, i)) ** 2
        return self.part(self.m, i).double(), self.part(self.v, i).double()

    def snapshot(self):
        return [(self.part(self.p, i).double(), self.part(self.g, i).double(), *self.state(i)) for i in range(len(self.sizes))]

    def outside(self):
        """What lies between the tensors, in every array."""
        keep = torch.ones(self.p.numel(), dtype=torch.bool, device="cuda")
        for i, n in enumerate(self.sizes):
            keep[self.at[i]:self.at[i] + n] = False
        return [t.float()[keep].clone() for t in (self.p, self.m, self.v, self.copy) if t is not None]

    def check(self, before, t, lr, gs=1.0):
        for i, (p, g, m, v) in enumerate(before):
            if p.numel() == 0:
                continue
            g = g * gs
            m1, v1 = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
            # the fp32 gradient scale and betas: relative u each, on top of the operations
            tm = 6 * U * ((B1 * m).abs() + ((1 - B1) * g).abs())
            tv = 8 * U * (B2 * v + (1 - B2) * g * g)
            root = v1.sqrt()
            step = lr / (1 - B1 ** t) * m1 / (root / (1 - B2 ** t) ** 0.5 + EPS)
            want = p * (1 - lr * self.decay[i]) - step
            tp = 3 * U * (p.abs() + want.abs()) + 16 * U * step.abs() + lr / (1 - B1 ** t) * tm / (root / (1 - B2 ** t) ** 0.5 + EPS)
            got = self.part(self.p, i)
            half = torch.finfo(got.dtype).eps / 2 if got.dtype == torch.bfloat16 else 0
            assert torch.all((got.double() - want).abs() <= tp + half * (want.abs() + tp)), i
            if self.copy is not None:
                assert torch.all((self.part(self.copy, i).double() - want).abs() <= tp + 2.0 ** -8 * (want.abs() + tp)), i
            gm, gv = self.state(i)
            if self.eight:
                ms, vs = self.scale(self.ms, i), self.scale(self.vs, i)
                blocks = -(-p.numel() // 128)
                for name, x, tol, s in (("m", m1.abs(), tm, ms), ("v", root, tv / (2 * root).clamp_min(1e-300), vs)):
                    pad = torch.nn.functional.pad(x, (0, blocks * 128 - x.numel())).view(blocks, 128).amax(1)
                    slack = torch.nn.functional.pad(tol, (0, blocks * 128 - x.numel())).view(blocks, 128).amax(1)
                    one = s[::128]
                    assert torch.all((one * 448 - pad).abs() <= slack + 2 * U * pad), (name, i)
                assert torch.all((gm - m1).abs() <= tm + (2.0 ** -4 + 4 * U) * m1.abs() + ms * 2.0 ** -10), i
                assert torch.all((gv.sqrt() - root).abs() <= tv / (2 * root).clamp_min(1e-300) + (2.0 ** -4 + 4 * U) * root + vs * 2.0 ** -9), i
                assert torch.all((gv > 0) | (root == 0) | (vs == 0)), i
            else:
                assert torch.all((gm - m1).abs() <= tm) and torch.all((gv - v1).abs() <= tv), i


SIZES = [[1], [10, 777], [128, 4096, 5000, 3], [100, 0, 257, 8192, 1], [100003]]


@pytest.mark.parametrize("offset", [0, 1, 4, 8])
@pytest.mark.parametrize("state", ["f32", "e4m3"])
@pytest.mark.parametrize("param,grad", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
def test_step(pk, param, grad, state, offset):
    for k, sizes in enumerate(SIZES):
        c = Case(pk, sizes, param, grad, state, offset=offset, seed=k, step=9, copy=k % 2 == 0)
        before, outside = c.snapshot(), c.outside()
        c.plan.step(1e-2)
        torch.cuda.synchronize()
        c.check(before, 10, 1e-2)
        for a, b in zip(outside, c.outside()):
            assert torch.equal(a, b)  # nothing between the tensors was written
        assert c.plan.get_step() == 10


@pytest.mark.parametrize("state", ["f32", "e4m3"])
def test_steps_from_zero(pk, state):
    """From empty states: every step against the states that the step before left."""
    c = Case(pk, [300, 5000, 64], state=state, fresh=True)
    for t in range(1, 6):
        before = c.snapshot()
        c.plan.step(1e-3)
        torch.cuda.synchronize()
        c.check(before, t, 1e-3)
        c.g.mul_(-0.7)


def test_scales_on_the_device(pk):
    c = Case(pk, [1000, 77], step=3)
    s = torch.tensor([0.5, 0.25], device="cuda")
    before = c.snapshot()
    c.plan.step(2e-2, grad_scale=2.0, scales=s.data_ptr())
    torch.cuda.synchronize()
    c.check(before, 4, 1e-2, gs=0.5)


def test_zero_gradients_and_tiny_states(pk):
    """No division by zero, and a block whose largest value is below 2^-100 is empty."""
    c = Case(pk, [256], state="e4m3", fresh=True, decay=0.0)
    c.g.zero_()
    p = c.p.clone()
    c.plan.step(1.0)
    assert torch.equal(c.p, p) and torch.all(c.ms[:2] == 0) and torch.all(c.vs[:2] == 0)
    c.g[:128] = 1e-36
    c.plan.step(1.0)
    assert float(c.ms[0]) == 0 and torch.all(c.m.float()[:256] == 0) and torch.all(torch.isfinite(c.p))


def test_a_small_root_stays_above_zero(pk):
    c = Case(pk, [128], state="e4m3", fresh=True)
    c.g.fill_(1e-12)
    c.g[c.at[0]] = 1.0
    c.plan.step(1e-3)
    v = c.part(c.v, 0).float()
    assert float(v[0]) == 448 and torch.all(v[1:] == 2.0 ** -9)


def test_nonfinite_gradients(pk):
    """A NaN or infinity stays where it is with fp32 states, and shows in the scale of its block with 8-bit ones."""
    c = Case(pk, [512])
    c.g[5], c.g[200] = float("nan"), float("inf")
    c.plan.step(1e-3)
    bad = ~torch.isfinite(c.part(c.p, 0))
    assert bad.nonzero().flatten().tolist() == [5, 200]
    c = Case(pk, [512], state="e4m3")
    c.g[5], c.g[200] = float("nan"), float("inf")
    c.plan.step(1e-3)
    assert torch.isfinite(c.ms[:4]).tolist() == [False, False, True, True]
    assert torch.isfinite(c.vs[:4]).tolist() == [False, False, True, True]


def test_tensors_without_gradient(pk):
    c = Case(pk, [300, 200, 5000])
    c.plan.set_grads([c.g[c.at[0]:].data_ptr(), None, c.g[c.at[2]:].data_ptr()])
    before = c.snapshot()
    c.plan.step(1e-2)
    torch.cuda.synchronize()
    assert torch.equal(c.part(c.p, 1).double(), before[1][0]) and torch.equal(c.state(1)[0], before[1][2])
    before[1] = tuple(t[:0] for t in before[1])
    c.check(before, 1, 1e-2)
    with pytest.raises(ValueError):
        c.plan.set_grads([None])


def test_no_tensors(pk):
    plan = pk.AdamW([])
    plan.step(1e-3)
    assert plan.get_step() == 1
    plan.set_step(41)
    plan.step(1e-3)
    assert plan.get_step() == 42


def test_many_tensors(pk):
    c = Case(pk, [1 + 37 * i % 900 for i in range(700)], state="e4m3")
    before = c.snapshot()
    c.plan.step(1e-2)
    torch.cuda.synchronize()
    c.check(before, 1, 1e-2)


@pytest.mark.parametrize("state", ["f32", "e4m3"])
def test_graph_replay_counts_steps(pk, state):
    a, b = Case(pk, [70000, 5], state=state, seed=3), Case(pk, [70000, 5], state=state, seed=3)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        a.plan.step(1e-2, stream=st.cuda_stream)
    for _ in range(4):
        g.replay()
        b.plan.step(1e-2)
    torch.cuda.synchronize()
    assert a.plan.get_step() == b.plan.get_step() == 4
    for x, y in ((a.p, b.p), (a.m, b.m), (a.v, b.v), (a.copy, b.copy)):
        assert torch.equal(x.float(), y.float())


def test_state_from_a_long_run(pk):
    """The device's running powers of beta agree with the closed form after set_step and after many steps."""
    c = Case(pk, [64], step=0, fresh=True)
    for _ in range(300):
        c.plan.step(1e-3)
    before = c.snapshot()
    c.plan.step(1e-3)
    torch.cuda.synchronize()
    c.check(before, 301, 1e-3)


def test_refusals(pk):
    t = torch.zeros(4, 256, device="cuda")
    host = torch.zeros(256)
    ok = dict(param=t[0].data_ptr(), grad=t[1].data_ptr(), m=t[2].data_ptr(), v=t[3].data_ptr(), n=256)
    for kw, word, opts in [(dict(param=None), "needs param", {}), (dict(n=-1), "values", {}), (dict(m=t[2].data_ptr() + 2), "aligned", {}),
                           (dict(grad=host.data_ptr()), "not device memory", {}), ({}, "m_scale", dict(state_dtype="e4m3")),
                           ({}, "betas", dict(beta1=1.0)), ({}, "eps", dict(eps=-1.0)), ({}, "step", dict(step=-1)), ({}, "out of range", dict(device=63))]:
        with pytest.raises(pk.PktError, match=word):
            pk.AdamW([pk.AdamWTensor(**{**ok, **kw})], **opts)
    plan = pk.AdamW([pk.AdamWTensor(**ok)])
    with pytest.raises(pk.PktError, match="not device memory"):
        plan.step(1e-3, scales=host.data_ptr())
    with pytest.raises(pk.PktError, match="not device memory"):
        plan.set_grads([host.data_ptr()])
    with pytest.raises(pk.PktError):
        plan.set_step(-1)
    with pytest.raises(pk.PktError, match="too many"):
        pk.AdamW([pk.AdamWTensor(**{**ok, "n": (1 << 63) - 1})])


def test_refuses_overlapping_arrays(pk):
    """What a step writes twice, or writes while it is another chunk's gradient, would depend on timing."""
    t = torch.zeros(8, 256, device="cuda")
    at = [t[i].data_ptr() for i in range(8)]
    ok = dict(param=at[0], grad=at[1], m=at[2], v=at[3], n=256)
    other = dict(param=at[4], grad=at[1], m=at[5], v=at[6], n=256)  # a shared gradient
    plan = pk.AdamW([pk.AdamWTensor(**ok), pk.AdamWTensor(**other)])
    for kw in (dict(param=at[0]), dict(m=at[0] + 1020), dict(v=at[2]), dict(copy_bf16=at[3] + 512), dict(n=257)):
        with pytest.raises(pk.PktError, match="writes overlap"):
            pk.AdamW([pk.AdamWTensor(**ok), pk.AdamWTensor(**{**other, **kw})])
    for g in (at[0], at[0] - 4, at[6] + 1020):
        with pytest.raises(pk.PktError, match="grad of tensor 1 overlaps"):
            pk.AdamW([pk.AdamWTensor(**ok), pk.AdamWTensor(**{**other, "grad": g})])
        with pytest.raises(pk.PktError, match="grad of tensor 1 overlaps"):
            plan.set_grads([at[1], g])
    plan.set_grads([at[7], None])
    t[7] = 1.0
    plan.step(1e-2)
    assert torch.all(t[2] != 0) and torch.all(t[5] == 0)
    pk.AdamW([pk.AdamWTensor(**ok), pk.AdamWTensor(**{**ok, "n": 0, "grad": at[0] + 8})])  # nothing is written twice


def test_gradients_stay_as_they_were_inside_a_capture(pk):
    c = Case(pk, [3000])
    before = c.snapshot()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        with pytest.raises(pk.PktError, match="stream capture"):
            c.plan.set_grads([None], st.cuda_stream)
        c.plan.step(1e-2, stream=st.cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    c.check(before, 1, 1e-2)


def test_a_plan_may_be_dropped_while_a_stream_is_captured(pk):
    a, b = Case(pk, [3000]), Case(pk, [500])
    before = a.snapshot()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        a.plan.step(1e-2, stream=st.cuda_stream)
        b.plan.close()
    g.replay()
    torch.cuda.synchronize()
    a.check(before, 1, 1e-2)


def test_two_plans_on_two_streams(pk):
    a, b = Case(pk, [300000, 7], seed=1), Case(pk, [200000], state="e4m3", seed=2)
    want = a.snapshot(), b.snapshot()
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    a.plan.step(1e-2, stream=s.cuda_stream)
    b.plan.step(1e-2, stream=t.cuda_stream)
    torch.cuda.synchronize()
    a.check(want[0], 1, 1e-2)
    b.check(want[1], 1, 1e-2)


@pytest.mark.parametrize("state", ["f32", "e4m3"])
def test_tensors_without_values_claim_nothing(pk, state):
    """Scales packed at ceil(n / 128) each: an empty tensor's arrays begin where the next one's do."""
    sizes, eight = [256, 0, 300, 0, 5], state == "e4m3"
    at = [sum(sizes[:i]) for i in range(5)]
    blocks = [-(-n // 128) for n in sizes]
    sat = [sum(blocks[:i]) for i in range(5)]
    p, m, v = torch.full((561,), 0.5, device="cuda"), torch.zeros(561, device="cuda"), torch.zeros(561, device="cuda")
    if eight:
        m, v = m.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
    g, ms, vs = torch.full((561,), 0.25, device="cuda"), torch.zeros(6, device="cuda"), torch.zeros(6, device="cuda")
    rec = [pk.AdamWTensor(param=p[a:].data_ptr(), grad=g[a:].data_ptr(), m=m[a:].data_ptr(), v=v[a:].data_ptr(), n=n,
                          m_scale=ms[b:].data_ptr() if eight else None, v_scale=vs[b:].data_ptr() if eight else None)
           for a, b, n in zip(at, sat, sizes)]
    plan = pk.AdamW(rec, state_dtype=state, eps=1e-8)
    plan.step(0.125)
    # a first step from empty states moves by lr m / (1 - b1) / (|g| + eps) = lr, 16 u of the step and 3 u of the value off
    assert torch.all((p.double() - 0.375).abs() <= 16 * U * 0.125 + 3 * U * 0.5 + 0.125 * 1e-8 / 0.25)
    if eight:
        assert torch.all(ms > 0) and torch.all(vs > 0)


def test_a_tensor_without_values_may_name_anything(pk):
    """No pointer of it is looked at: host memory, an odd address, one that another tensor writes."""
    t = torch.zeros(4, 256, device="cuda")
    host = torch.zeros(256)
    ok = dict(param=t[0].data_ptr(), grad=t[1].data_ptr(), m=t[2].data_ptr(), v=t[3].data_ptr(), n=256)
    for kw in (dict(param=host.data_ptr()), dict(m=t[2].data_ptr() + 1), dict(v=t[0].data_ptr()), dict(grad=t[1].data_ptr() + 3), dict(copy_bf16=host.data_ptr())):
        plan = pk.AdamW([pk.AdamWTensor(**ok), pk.AdamWTensor(**{**ok, "n": 0, **kw})])
        plan.set_grads([t[1].data_ptr(), t[1].data_ptr() + 1])
        plan.step(1e-3)
    torch.cuda.synchronize()
    assert torch.all(t == 0)


def test_the_step_is_not_read_inside_a_capture(pk):
    """Refused before anything is enqueued, so the capture goes on."""
    c = Case(pk, [3000])
    before = c.snapshot()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        with pytest.raises(pk.PktError, match="stream capture"):
            c.plan.get_step(st.cuda_stream)
        c.plan.step(1e-2, stream=st.cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    c.check(before, 1, 1e-2)
    assert c.plan.get_step() == 1
