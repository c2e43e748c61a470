"""The AdamW step against its formula.

m and v are rounded to fp32 at every operation as it is written, so the same operations
of torch give the same bits, and the same codes in 8 bits.  The change of p is off by at
most 2^-19 of itself (approximate root and quotient, 2^-21 each, and fewer than eight
roundings), and p is rounded twice.  Against 64 bits m and v are off by their roundings: at
most 4 2^-24 of their terms.
"""
import math

import pytest
import torch

import rows_reference as ref
from expert_reference import close

pytestmark = pytest.mark.gpu
RULE = dict(lr=2e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.05)
SIZES = {"one": [1], "blocks": [255, 256, 257, 2048, 2049], "empty among": [0, 300, 0], "many": [1 + 37 * i % 700 for i in range(900)],
         "large": [3_000_001, 70_000]}


def _to_codes(v):
    n = v.numel()
    blocks = torch.nn.functional.pad(v.reshape(-1), (0, -n % 256)).view(-1, 256)
    scale = blocks.abs().amax(1) / torch.full((), 448.0, device=v.device)
    codes = (blocks / torch.where(scale > 0, scale, 1.0)[:, None]).to(torch.float8_e4m3fn)
    return codes.view(-1)[:n], scale


def _of_codes(codes, scale):
    return codes.reshape(-1).float() * scale.repeat_interleave(256)[:codes.numel()]


class Plain:
    """The step in torch operations, each rounded to fp32."""

    def __init__(self, params, bits, master):
        self.p = [p.detach().clone() for p in params]
        self.master = [p.float() if master and p.dtype != torch.float32 else None for p in self.p]
        self.bits = bits
        self.m = [torch.zeros(p.numel(), device=p.device) for p in self.p]
        self.v = [torch.zeros(p.numel(), device=p.device) for p in self.p]
        self.off = [torch.zeros(p.numel(), device=p.device) for p in self.p]  # bound of p's error in one step
        self.t = 0

    def follow(self, params, state):
        """Compares the parameters, and goes on from them."""
        for i, p in enumerate(params):
            mine, off = self.p[i].reshape(-1), self.off[i].double()
            if self.master[i] is not None:
                close(state.master[i].reshape(-1), self.master[i].reshape(-1).double(), off, (i, "master"))
                assert torch.equal(p, state.master[i].to(p.dtype))
                self.master[i] = state.master[i].clone()
            else:  # rounded to its own type: one step further where the two lie on both sides of a border
                u = 0 if p.dtype == torch.float32 else ref.U[p.dtype]
                close(p.reshape(-1), mine.double(), off + 2 * u * mine.double().abs() + 2 * (u > 0) * ref.FLOOR[p.dtype], (i, "parameter"))
            self.p[i] = p.clone()

    def step(self, grads, lr, betas, eps, weight_decay, factor=1.0):
        self.t += 1
        rate, root = lr / (1 - betas[0] ** self.t), math.sqrt(1 - betas[1] ** self.t)
        keep = 1 - lr * weight_decay

        def f32(v):
            return torch.tensor(v, dtype=torch.float64).float().to(self.p[0].device)

        factor, rate, root = f32(factor), f32(rate), f32(root)
        for i, g in enumerate(grads):
            if g.numel() == 0:
                continue
            p = (self.p[i] if self.master[i] is None else self.master[i]).reshape(-1).float()
            g = g.reshape(-1).float() * factor
            m = self.m[i] * betas[0] + g * (1 - betas[0])
            v = self.v[i] * betas[1] + (g * g) * (1 - betas[1])
            change = (m / (v.sqrt() / root + eps)) * rate
            p = p * keep - change
            self.off[i] = 2.0 ** -19 * change.abs() + 3 * ref.E32 * p.abs()
            if self.bits == 8:
                m = _of_codes(*_to_codes(m))
                codes, scale = _to_codes(v.sqrt())
                codes = torch.where((v > 0) & (codes.float() == 0), torch.full_like(codes.float(), 2.0 ** -9), codes.float())
                v = _of_codes(codes, scale).square()
            self.m[i], self.v[i] = m, v
            if self.master[i] is not None:
                self.master[i] = p.view(self.p[i].shape)
            self.p[i] = p.to(self.p[i].dtype).view(self.p[i].shape)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                   (torch.bfloat16, torch.float32), (torch.float16, torch.float16), "mixed"])
def test_steps_equal_the_written_operations(hb, cuda, sizes, types, bits):
    gen = torch.Generator(device=cuda).manual_seed(len(sizes) + bits)
    n = SIZES[sizes]
    of = [types if types != "mixed" else [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)][i % 3]
          for i in range(len(n))]

    def normal(size, dtype, scale):
        return (torch.randn(size, generator=gen, device=cuda) * scale).to(dtype)

    for master in (False, True):
        params = [normal(k, t[0], 0.5) for k, t in zip(n, of)]
        state = hb.adamw_state(params, bits=bits, master=master)
        plain = Plain(params, bits, master)
        for turn in range(3):
            grads = [normal(k, t[1], 0.01 * 3 ** turn) for k, t in zip(n, of)]
            before = [g.clone() for g in grads]
            norm, limit = hb.grad_norm(grads), [None, 0.05, 1e6][turn]
            factor = 1.0 if limit is None else min(1.0, limit / (float(norm) + 1e-6))
            hb.adamw_step(params, grads, state, **RULE, norm=None if limit is None else norm, max_norm=limit)
            plain.step(grads, **RULE, factor=factor)
            plain.follow(params, state)
            assert int(state.step) == turn + 1
            assert all(torch.equal(g, b) for g, b in zip(grads, before))
        m, v = hb.adamw_moments(state)
        for i in range(len(params)):
            assert torch.equal(m[i].view(-1), plain.m[i]) and torch.equal(v[i].view(-1), plain.v[i]), (i, "moments")


def test_against_64_bits(hb, cuda):
    gen = torch.Generator(device=cuda).manual_seed(1)
    p = torch.randn(5000, generator=gen, device=cuda)
    state = hb.adamw_state([p])
    p64, m, v = p.double(), torch.zeros(5000, dtype=torch.float64, device=cuda), torch.zeros(5000, dtype=torch.float64, device=cuda)
    b1, b2 = RULE["betas"]
    sum_m, change = torch.zeros_like(m), torch.zeros_like(m)
    for t in range(1, 6):
        g = torch.randn(5000, generator=gen, device=cuda) * 0.1
        hb.adamw_step([p], [g], state, **RULE)
        g64 = g.double()
        m, v = b1 * m + (1 - b1) * g64, b2 * v + (1 - b2) * g64 ** 2
        sum_m = b1 * sum_m + (1 - b1) * g64.abs()
        by = v.sqrt() / math.sqrt(1 - b2 ** t) + RULE["eps"]
        p64 = p64 * (1 - RULE["lr"] * RULE["weight_decay"]) - RULE["lr"] / (1 - b1 ** t) * m / by
        change = change + 4 * t * ref.E32 * RULE["lr"] / (1 - b1 ** t) * sum_m / by + (2.0 ** -19 + 4 * t * ref.E32) * RULE["lr"] / (1 - b1 ** t) * m.abs() / by \
            + 2 * ref.E32 * p64.abs()
        close(state.exp_avg[0], m, 4 * t * ref.E32 * sum_m, "m")
        close(state.exp_avg_sq[0], v, 5 * t * ref.E32 * v, "v")
        close(p, p64, change + 2 * ref.E32 * p64.abs(), "p")


def test_views_and_strides(hb, cuda):
    """Parameters off the 16-byte grid, transposed, scalars; a state of either kind."""
    gen = torch.Generator(device=cuda).manual_seed(2)
    flat = torch.randn(4000, generator=gen, device=cuda).to(torch.bfloat16)
    params = [flat[1:1001].view(10, 100), flat[1001:2001].view(50, 20).t(), flat[2003], flat[2016:2016 + 600]]
    grads = [torch.randn(p.shape, generator=gen, device=cuda).to(torch.bfloat16) for p in params]
    grads[1] = grads[1].t().contiguous().t()
    for bits in (8, 32):
        mine, dense = [p.clone() for p in params], [p.clone() for p in params]
        buffer = flat.clone()
        views = [buffer[1:1001].view(10, 100), buffer[1001:2001].view(50, 20).t(), buffer[2003], buffer[2016:2616]]
        mine[1] = mine[1].t().contiguous().t()
        dense[1] = dense[1].t().contiguous()
        dense_grads = [g.t() if i == 1 else g for i, g in enumerate(grads)]
        states = [hb.adamw_state(v, bits=bits, master=True) for v in (mine, dense, views)]
        for _ in range(2):
            hb.adamw_step(mine, grads, states[0], **RULE)
            hb.adamw_step(dense, dense_grads, states[1], **RULE)
            hb.adamw_step(views, grads, states[2], **RULE)
        for a, b, c in zip(mine, dense, views):
            assert torch.equal(a, c) and torch.equal(a, b if a.shape == b.shape else b.t())
        kept = torch.ones(4000, dtype=torch.bool, device=cuda)
        kept[1:2001] = kept[2003] = kept[2016:2616] = False
        assert torch.equal(buffer[kept], flat[kept])


def test_small_second_moments_are_kept(hb, cuda):
    """Next to one large gradient in a block, small ones keep the smallest code: a later step stays finite and small."""
    p = torch.zeros(256, device=cuda)
    g = torch.full((256,), 1e-12, device=cuda)
    g[0] = 1.0
    state = hb.adamw_state([p], bits=8)
    hb.adamw_step([p], [g], state, **RULE)
    m, v = hb.adamw_moments(state)
    assert bool((v[0] > 0).all())
    for _ in range(3):
        hb.adamw_step([p], [torch.zeros_like(g)], state, **RULE)
    # m / sqrt(v) of a first step is sqrt(1 - b2) / (1 - b1) less than 1 without the bias corrections, and only shrinks
    assert bool(torch.isfinite(p).all()) and float(p.abs().max()) <= 4 * 1.01 * RULE["lr"] * math.sqrt(1 / (1 - 0.98)) * 0.2


def test_not_a_number(hb, cuda):
    for bits in (32, 8):
        p = [torch.ones(600, device=cuda), torch.ones(300, device=cuda)]
        state = hb.adamw_state(p, bits=bits)
        g = [torch.ones(600, device=cuda), torch.ones(300, device=cuda)]
        g[0][300] = math.nan
        hb.adamw_step(p, g, state, **RULE)
        assert bool(torch.isnan(p[0][300])) and int(torch.isnan(p[0]).sum()) == 1 and bool(torch.isfinite(p[1]).all())
        m, _ = hb.adamw_moments(state)
        assert bool(torch.isfinite(m[0][:256]).all()) and bool(torch.isnan(m[0][300]))
        hb.adamw_step(p, g, state, **RULE, norm=hb.grad_norm(g), max_norm=1.0)
        assert all(bool(torch.isnan(v).all()) for v in p)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(hb, cuda, bits):
    """A captured step replayed: the count, the rate and the norm are read anew."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    sizes = [5000, 77]
    p = [torch.randn(n, generator=gen, device=cuda) for n in sizes]
    q = [v.clone() for v in p]
    g = [torch.randn(n, generator=gen, device=cuda) for n in sizes]
    a, b = hb.adamw_state(p, bits=bits), hb.adamw_state(q, bits=bits)
    rate = torch.tensor(1e-3, device=cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hb.adamw_step(p, g, a, lr=rate, norm=hb.grad_norm(g), max_norm=1.0)
    for turn in range(4):
        for v in g:
            v.normal_(generator=gen)
        rate.fill_(1e-3 * (turn + 1))
        graph.replay()
        hb.adamw_step(q, g, b, lr=float(rate), norm=hb.grad_norm(g), max_norm=1.0)
        assert int(a.step) == int(b.step) == turn + 1
        assert all(torch.equal(x, y) for x, y in zip(p, q))


def test_written_and_refused(hb, cuda):
    p, g = torch.ones(600, device=cuda), torch.ones(600, device=cuda)
    state = hb.adamw_state([p], bits=8, master=True)
    versions = [t._version for t in (p, state.exp_avg[0], state.exp_avg_scale[0], state.step, g)]
    hb.adamw_step([p], [g], state, lr=0.0)
    now = [t._version for t in (p, state.exp_avg[0], state.exp_avg_scale[0], state.step, g)]
    assert all(a < b for a, b in zip(versions[:4], now[:4])) and versions[4] == now[4] and state.master == [None]
    s32 = hb.adamw_state([p])
    kept = p.clone()
    flat = torch.ones(1000, device=cuda)
    half = p.half()
    for call in (lambda: hb.adamw_step([], [], state, lr=0.1), lambda: hb.adamw_step([p], [], state, lr=0.1), lambda: hb.adamw_step([p], [g[:5]], s32, lr=0.1),
                 lambda: hb.adamw_step([p], [g.half()], s32, lr=0.1), lambda: hb.adamw_step([p], [g.double()], s32, lr=0.1),
                 lambda: hb.adamw_step([p], [g.cpu()], s32, lr=0.1), lambda: hb.adamw_step([p], [p], s32, lr=0.1),
                 lambda: hb.adamw_step([flat[:600]], [flat[300:900]], s32, lr=0.1), lambda: hb.adamw_step([p, p], [g, g], hb.adamw_state([p, p]), lr=0.1),
                 lambda: hb.adamw_step([p], [g], s32, lr=-1.0), lambda: hb.adamw_step([p], [g], s32, lr=0.1, betas=(1.0, 0.9)),
                 lambda: hb.adamw_step([p], [g], s32, lr=0.1, eps=-1.0), lambda: hb.adamw_step([p], [g], s32, lr=0.1, weight_decay=math.nan),
                 lambda: hb.adamw_step([p], [g], s32, lr=0.1, max_norm=1.0), lambda: hb.adamw_step([p], [g], s32, lr=0.1, norm=hb.grad_norm([g])),
                 lambda: hb.adamw_step([p], [g], s32, lr=torch.ones(2, device=cuda)), lambda: hb.adamw_step([p], [g], s32._replace(step=s32.step.long()), lr=0.1),
                 lambda: hb.adamw_step([p], [g], s32._replace(exp_avg=state.exp_avg), lr=0.1),
                 lambda: hb.adamw_step([p], [g], state._replace(exp_avg_scale=[g]), lr=0.1),
                 lambda: hb.adamw_step([half], [g], hb.adamw_state([half])._replace(master=[half]), lr=0.1),
                 lambda: hb.adamw_state([p], bits=4), lambda: hb.adamw_state([])):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(p, kept) and int(s32.step) == 0
