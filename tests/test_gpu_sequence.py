"""The sequence operators (turbompc_b200.sequence) against their definitions in
64 bits: linear attention as its token-by-token recurrence, the residual norm
and the gated linear layer as written, gradients by autograd of those forms and
by central differences of the operators themselves.

Errors are norm-wise, |got - want| / |want|.  Tolerances:
* bfloat16 results: the stored value is rounded once (at most 2^-9 of each
  element), and at most three factors inside a product of sums are rounded to
  bfloat16 on the way, each at most 2^-9 norm-wise: 4 * 2^-9;
* float32 results (states included, whatever the inputs' type): sums of at
  most 2^12 terms, and factors split into two bfloat16 terms, 2^-17 each; with
  a factor of four: 2^-15;
* the norm in float32: a few roundings and a sum of at most 2^14 squares: 2^-20;
* dlog_decay: a sum of signed terms over every token, so its error is taken
  against the root sum of squares of the sequences' shares: 2^-12."""
import math

import pytest
import torch

from turbompc_b200 import sequence

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
F32_TOL = 2.0 ** -15
TOL = {torch.float32: F32_TOL, torch.bfloat16: 4 * 2.0 ** -9}
DLOG_TOL = 2.0 ** -12


def err(got, want):
    want = want.double()
    n = want.norm()
    return float((got.double() - want).norm() / (n if n > 0 else 1.0))


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ref_attention(q, k, v, log_decay, initial=None, lengths=None, scale=None):
    """S_t = d S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t, one token at a time, 64 bits."""
    B, T, H, dk = q.shape
    rep = H // k.shape[2]
    scale = dk ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double().repeat_interleave(rep, 2), v.double().repeat_interleave(rep, 2)
    d = torch.exp(log_decay.double())[None, :, None, None]
    S = torch.zeros(B, H, dk, v.shape[-1], dtype=torch.float64, device=q.device) if initial is None else initial.double()
    out = []
    for t in range(T):
        new = d * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        o = scale * (q[:, t, :, :, None] * new).sum(2)
        if lengths is not None:
            on = (t < lengths)[:, None, None]
            new = torch.where(on[..., None], new, S)
            o = torch.where(on, o, torch.zeros_like(o))
        S = new
        out.append(o)
    o = torch.stack(out, 1) if out else torch.zeros(B, 0, H, v.shape[-1], dtype=torch.float64, device=q.device)
    return o, S


def attention_inputs(B, T, H, G, dk, dv, dtype, seed, state=True, lengths=None):
    g = gen(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    q, k, v = n(B, T, H, dk).to(dtype), n(B, T, G, dk).to(dtype), n(B, T, G, dv).to(dtype)
    i = 2.0 + 5.0 * torch.arange(H, device="cuda") / max(H - 1, 1)
    log_decay = torch.log1p(-torch.exp2(-i))
    S = 2 * n(B, H, dk, dv) if state else None
    L = None
    if lengths == "ragged":
        L = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        L[0] = 0
        if B > 1:
            L[1] = T
        if B > 2:
            L[2] = min(1, T)
    return q, k, v, log_decay, S, L


SHAPES = [
    # B, T, H, G, dk, dv
    (1, 1, 1, 1, 1, 1),
    (3, 1, 2, 1, 16, 16),
    (2, 15, 2, 2, 32, 24),
    (3, 16, 4, 2, 32, 32),
    (2, 17, 3, 1, 20, 50),
    (2, 63, 4, 4, 64, 64),
    (2, 64, 2, 2, 64, 64),
    (3, 65, 4, 2, 48, 64),
    (5, 61, 4, 4, 64, 64),
    (2, 127, 2, 1, 128, 128),
    (2, 129, 4, 1, 128, 80),
    (2, 200, 2, 2, 7, 128),
    (1, 301, 8, 4, 64, 64),
    (1, 1000, 2, 1, 96, 128),
    (1, 2049, 1, 1, 64, 32),
    (300, 5, 2, 1, 32, 32),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("lengths", [None, "ragged"])
def test_linear_attention_forward(shape, dtype, lengths):
    q, k, v, g, S, L = attention_inputs(*shape, dtype, 1, state=shape[1] % 2 == 1, lengths=lengths)
    o, state = sequence.linear_attention(q, k, v, g, initial_state=S, lengths=L, return_state=True)
    ro, rs = ref_attention(q, k, v, g, S, L)
    assert o.dtype == dtype and state.dtype == torch.float32
    assert err(o, ro) < TOL[dtype]
    assert err(state, rs) < F32_TOL
    assert torch.equal(o, sequence.linear_attention(q, k, v, g, initial_state=S, lengths=L))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("lengths", [None, "ragged"])
def test_linear_attention_backward(shape, dtype, lengths):
    with_state = shape[1] % 2 == 1
    q, k, v, g, S, L = attention_inputs(*shape, dtype, 2, state=with_state, lengths=lengths)
    gn = gen(3)
    do = torch.randn(shape[0], shape[1], shape[2], shape[5], generator=gn, device="cuda").to(dtype)
    dS = torch.randn(shape[0], shape[2], shape[4], shape[5], generator=gn, device="cuda") if with_state else None
    leaves = [t.requires_grad_(True) for t in (q, k, v, g, S) if t is not None]
    o, state = sequence.linear_attention(q, k, v, g, initial_state=S, lengths=L, return_state=True)
    if with_state:
        got = torch.autograd.grad([o, state], leaves, [do, dS])
    else:
        got = torch.autograd.grad(o, leaves, do)
    # a decay per sequence, so that the shares of dlog_decay are known
    B = shape[0]
    refs = [t.detach().double().requires_grad_(True) for t in leaves]
    gb = g.detach().double()[None].repeat(B, 1).requires_grad_(True)
    parts = []
    for b in range(B):
        sl = slice(b, b + 1)
        parts.append(ref_attention(refs[0][sl], refs[1][sl], refs[2][sl], gb[b], refs[4][sl] if with_state else None,
                                   None if L is None else L[sl]))
    ro, rs = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
    loss = (ro * do.double()).sum() + ((rs * dS.double()).sum() if with_state else 0)
    want = torch.autograd.grad(loss, [refs[0], refs[1], refs[2], gb] + ([refs[4]] if with_state else []))
    for i, name in enumerate(("dq", "dk", "dv")):
        assert got[i].dtype == dtype
        assert err(got[i], want[i]) < TOL[dtype], name
    scale = want[3].pow(2).sum(0).sqrt()
    assert float(((got[3].double() - want[3].sum(0)).abs() / scale.clamp(min=1e-30)).max()) < DLOG_TOL
    if with_state:
        assert err(got[4], want[4]) < F32_TOL


@pytest.mark.parametrize("shape", [(1250, 5, 2, 1, 16, 24), (610, 3, 1, 1, 64, 40), (155, 4, 2, 1, 128, 20)], ids=str)
@pytest.mark.parametrize("lengths", [None, "ragged"])
def test_linear_attention_backward_of_many_states(shape, lengths):
    """More float states than the device holds at once: the gradient's passes one after the other."""
    test_linear_attention_backward(shape, torch.float32, lengths)


def test_linear_attention_backward_of_the_state_alone():
    q, k, v, g, S, _ = attention_inputs(2, 33, 2, 1, 32, 32, torch.float32, 4)
    leaves = [t.requires_grad_(True) for t in (q, k, v, g, S)]
    _, state = sequence.linear_attention(q, k, v, g, initial_state=S, return_state=True)
    dS = torch.randn(state.shape, generator=gen(5), device="cuda")
    got = torch.autograd.grad(state, leaves, dS)
    refs = [t.detach().double().requires_grad_(True) for t in leaves]
    _, rs = ref_attention(*refs)
    want = torch.autograd.grad(rs, refs, dS.double(), allow_unused=True)
    assert not got[0].any()
    for i in (1, 2, 4):
        assert err(got[i], want[i]) < F32_TOL
    assert err(got[3], want[3]) < DLOG_TOL


def test_linear_attention_gradient_against_differences():
    """o is linear in each of q, k, v and the state, so a central difference
    along the gradient has no truncation error there; in log_decay a step of
    2^-7 leaves (2^-7 T)^2 / 6 relative at worst, 1 % for T = 33."""
    q, k, v, g, S, L = attention_inputs(2, 33, 4, 2, 32, 16, torch.float32, 6, lengths="ragged")
    w = torch.randn(2, 33, 4, 16, generator=gen(7), device="cuda")
    base = [q, k, v, g, S]

    def loss(xs):
        with torch.no_grad():
            return (sequence.linear_attention(*xs[:4], initial_state=xs[4], lengths=L).double() * w).sum()

    leaves = [t.clone().requires_grad_(True) for t in base]
    got = torch.autograd.grad(sequence.linear_attention(*leaves[:4], initial_state=leaves[4], lengths=L), leaves, w)
    for i, gi in enumerate(got):
        step = 2.0 ** -7 if i == 3 else 1.0
        d = gi / gi.abs().max()
        hi = loss([t + step * d if j == i else t for j, t in enumerate(base)])
        lo = loss([t - step * d if j == i else t for j, t in enumerate(base)])
        want = (gi.double() * d).sum()
        assert abs(float((hi - lo) / (2 * step) - want)) < (1e-2 if i == 3 else 1e-4) * abs(float(want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_attention_strided_inputs(dtype):
    """q, k, v as slices of one projection, heads-first views, an odd base
    address, a broadcast batch, and a last axis that is not contiguous."""
    B, T, H, D = 2, 37, 4, 32
    g = gen(8)
    log_decay = attention_inputs(B, T, H, H, D, D, dtype, 0)[3]
    qkv = torch.randn(B, T, 3, H, D, generator=g, device="cuda").to(dtype)
    cases = [tuple(qkv[:, :, i] for i in range(3))]
    cases.append(tuple(torch.randn(B, H, T, D, generator=g, device="cuda").to(dtype).transpose(1, 2) for _ in range(3)))
    odd = torch.randn(3, B * T * H * D + 1, generator=g, device="cuda").to(dtype)
    cases.append(tuple(odd[i, 1:].view(B, T, H, D) for i in range(3)))
    cases.append(tuple(torch.randn(1, T, H, D, generator=g, device="cuda").to(dtype).expand(B, T, H, D) for _ in range(3)))
    cases.append(tuple(torch.randn(B, T, D, H, generator=g, device="cuda").to(dtype).transpose(2, 3) for _ in range(3)))
    cases.append(tuple(torch.randn(B, T, H, D + 1, generator=g, device="cuda").to(dtype)[..., :D] for _ in range(3)))
    for q, k, v in cases:
        o = sequence.linear_attention(q, k, v, log_decay)
        want = sequence.linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), log_decay)
        assert err(o, ref_attention(q, k, v, log_decay)[0]) < TOL[dtype]
        assert err(o, want) < TOL[dtype]
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        do = torch.randn(o.shape, generator=g, device="cuda").to(dtype)
        for w_ in (do, do[:1].expand_as(do), do.transpose(1, 2).contiguous().transpose(1, 2)):
            got = torch.autograd.grad(sequence.linear_attention(*leaves, log_decay), leaves, w_)
            refs = [t.detach().double().requires_grad_(True) for t in leaves]
            ref = torch.autograd.grad(ref_attention(*refs, log_decay)[0], refs, w_.double())
            for a, b in zip(got, ref):
                assert err(a, b) < TOL[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_attention_ignores_what_lies_past_the_lengths(dtype):
    """NaN and infinities in q, k, v and do past a sequence's end reach nothing;
    lengths out of range are clamped."""
    q, k, v, g, S, _ = attention_inputs(4, 70, 2, 1, 64, 64, dtype, 9)
    L = torch.tensor([0, 1, 65, 70], dtype=torch.int32, device="cuda")
    do = torch.randn(4, 70, 2, 64, generator=gen(10), device="cuda").to(dtype)
    clean = [t.clone().requires_grad_(True) for t in (q, k, v, S)]
    o, st = sequence.linear_attention(*clean[:3], g, initial_state=clean[3], lengths=L, return_state=True)
    want = torch.autograd.grad(o, clean, do)
    dirty = [t.clone() for t in (q, k, v)]
    do2 = do.clone()
    for t in (*dirty, do2):
        for b in range(4):
            t[b, L[b]:] = float("nan") if b % 2 else float("inf")
    dirty = [t.requires_grad_(True) for t in (*dirty, S.clone())]
    L2 = torch.tensor([-5, 1, 65, 1000], dtype=torch.int32, device="cuda")
    o2, st2 = sequence.linear_attention(*dirty[:3], g, initial_state=dirty[3], lengths=L2, return_state=True)
    got = torch.autograd.grad(o2, dirty, do2)
    assert torch.equal(o, o2) and torch.equal(st, st2)
    assert not o2[0].any() and torch.equal(st2[0], S[0])
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_attention_extreme_decays(dtype):
    """log_decay 0 (a plain running sum), -inf (each token alone) and one whose
    power over a chunk underflows."""
    q, k, v, _, S, _ = attention_inputs(2, 130, 4, 4, 32, 32, dtype, 11)
    g = torch.tensor([0.0, float("-inf"), -50.0, -1e-6], device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v, S)]
    o, st = sequence.linear_attention(*leaves[:3], g, initial_state=S, return_state=True)
    ro, rs = ref_attention(q, k, v, g.clamp(min=-1e3), S)
    do = torch.randn(o.shape, generator=gen(12), device="cuda").to(dtype)
    got = torch.autograd.grad(o, leaves, do)
    refs = [t.detach().double().requires_grad_(True) for t in leaves]
    want = torch.autograd.grad(ref_attention(*refs[:3], g.clamp(min=-1e3), refs[3])[0], refs, do.double())
    for h in range(4):
        assert err(o[:, :, h], ro[:, :, h]) < TOL[dtype]
        assert err(st[:, h], rs[:, h]) < F32_TOL
        for a, b in zip(got[:3], want[:3]):
            assert err(a[:, :, h], b[:, :, h]) < TOL[dtype]
        assert err(got[3][:, h], want[3][:, h]) < F32_TOL


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_attention_offsets_past_32_bits(dtype):
    """Token strides of 2^30 elements: the third token lies past 2^31."""
    step, H, D = 2 ** 30, 2, 16
    buf = torch.empty(2 * step + 3 * H * D, dtype=dtype, device="cuda")
    q, k, v = (torch.as_strided(buf, (1, 3, H, D), (3 * H * D, step, D, 1), i * H * D) for i in range(3))
    for i, t in enumerate((q, k, v)):
        t.copy_(torch.randn(1, 3, H, D, generator=gen(13 + i), device="cuda"))
    g = torch.full((H,), -0.1, device="cuda")
    o, st = sequence.linear_attention(q, k, v, g, return_state=True)
    ro, rs = ref_attention(q, k, v, g)
    assert err(o, ro) < TOL[dtype] and err(st, rs) < F32_TOL


def test_linear_attention_empty():
    for B, T in ((0, 5), (2, 0)):
        q, k, v, g, S, _ = attention_inputs(B, T, 2, 1, 16, 8, torch.float32, 14)
        leaves = [t.requires_grad_(True) for t in (q, k, v, g, S)]
        o, st = sequence.linear_attention(q, k, v, g, initial_state=S, return_state=True)
        assert o.shape == (B, T, 2, 8) and torch.equal(st, S)
        got = torch.autograd.grad([o, st], leaves, [torch.ones_like(o), torch.ones_like(st)])
        assert not got[3].any() and torch.equal(got[4], torch.ones_like(S))
        o, st = sequence.linear_attention(q.detach(), k.detach(), v.detach(), g.detach(), return_state=True)
        assert not st.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_attention_is_reproducible_and_batch_independent(dtype):
    q, k, v, g, S, _ = attention_inputs(40, 150, 4, 2, 64, 64, dtype, 15)
    leaves = [t.requires_grad_(True) for t in (q, k, v, g, S)]
    do = torch.randn(40, 150, 4, 64, generator=gen(16), device="cuda").to(dtype)

    def once():
        o, st = sequence.linear_attention(q, k, v, g, initial_state=S, return_state=True)
        return [o, st, *torch.autograd.grad(o, leaves, do)]

    first = once()
    for _ in range(3):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,G,dk,dv", [(1, 1, 1, 1, 1), (3, 4, 2, 32, 32), (64, 4, 4, 32, 24), (5, 2, 1, 7, 50),
                                         (2, 3, 3, 128, 128), (9, 8, 1, 64, 63), (0, 2, 1, 16, 16)])
def test_step_matches_recurrence(B, H, G, dk, dv, dtype):
    q, k, v, g, S, _ = attention_inputs(B, 1, H, G, dk, dv, dtype, 17)
    ro, rs = ref_attention(q, k, v, g, S)
    out = torch.empty_like(S)
    before = S.clone()
    o = sequence.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, S, state_out=out)
    assert torch.equal(S, before)
    if B:
        assert err(o, ro[:, 0]) < TOL[dtype] and err(out, rs) < F32_TOL
    o2 = sequence.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, S)
    assert torch.equal(o, o2) and torch.equal(S, out)


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_continue_a_prompt(dtype):
    """A prompt, then single tokens (views of strided tensors), equal the whole sequence."""
    q, k, v, g, S, _ = attention_inputs(3, 80, 4, 2, 64, 48, dtype, 18)
    whole, end = sequence.linear_attention(q, k, v, g, initial_state=S, return_state=True)
    o, st = sequence.linear_attention(q[:, :70], k[:, :70], v[:, :70], g, initial_state=S, return_state=True)
    assert err(o, whole[:, :70]) < TOL[dtype]
    for t in range(70, 80):
        o = sequence.linear_attention_step(q[:, t], k[:, t], v[:, t], g, st)
        assert err(o, whole[:, t]) < TOL[dtype]
    assert err(st, end) < F32_TOL


def test_operators_run_on_the_current_stream():
    """Inputs made on another stream, work ordered by that stream alone."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q, k, v, g, S, _ = attention_inputs(64, 300, 4, 4, 64, 64, torch.bfloat16, 19)
        o, st = sequence.linear_attention(q, k, v, g, initial_state=S, return_state=True)
        y, t = sequence.add_rms_norm(o, q, torch.ones(64, device="cuda", dtype=torch.bfloat16))
        w = torch.randn(100, 64, generator=gen(20), device="cuda").bfloat16()
        h = sequence.gated_linear(y, w, w)
    side.synchronize()
    ro, _ = ref_attention(q, k, v, g, S)
    assert err(o, ro) < TOL[torch.bfloat16]
    p = y.double() @ w.double().t()
    assert err(h, p * torch.sigmoid(p) * p) < TOL[torch.bfloat16]


# ---------------------------------------------------------------------------
# Residual addition and norm
# ---------------------------------------------------------------------------
NORM_TOL = {torch.float32: 2.0 ** -20, torch.bfloat16: 4 * 2.0 ** -9}


def ref_norm(x, r, w, eps=1e-6):
    t = x.double() + (r.double() if r is not None else 0)
    return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps) * w.double(), t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 16), (7, 33), (64, 128), (300, 250), (5, 1000), (1000, 512), (3, 1024),
                                    (9, 1025), (4, 4096), (2, 4099), (3, 8192), (2, 16384), (5000, 20)])
@pytest.mark.parametrize("residual", [True, False])
def test_add_rms_norm(rows, d, dtype, residual):
    g = gen(21)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    x, r, w = n(rows, d), (n(rows, d) if residual else None), n(d)
    dy, ds = n(rows, d), n(rows, d)
    leaves = [t.requires_grad_(True) for t in (x, r, w) if t is not None]
    y, t = sequence.add_rms_norm(x, r, w)
    ry, rt = ref_norm(x, r, w)
    assert err(y, ry) < NORM_TOL[dtype] and err(t, rt) < NORM_TOL[dtype]
    refs = [z.detach().double().requires_grad_(True) for z in leaves]
    out = ref_norm(refs[0], refs[1] if residual else None, refs[-1])
    if residual:
        got = torch.autograd.grad([y, t], leaves, [dy, ds])
        want = torch.autograd.grad(out, refs, [dy.double(), ds.double()])
    else:
        got = torch.autograd.grad(y, leaves, dy)
        want = torch.autograd.grad(out[0], refs, dy.double())
    for a, b in zip(got, want):
        # dx of a single element is a difference of equal terms; it is compared on the scale of dy
        if float(b.norm()) > 1e-3 * float(dy.norm()):
            assert err(a, b) < (NORM_TOL[dtype] * 16 if dtype == torch.float32 else NORM_TOL[dtype])
    again = torch.autograd.grad(sequence.add_rms_norm(x, r, w)[0], leaves, dy)
    for a, b in zip(again, torch.autograd.grad(sequence.add_rms_norm(x, r, w)[0], leaves, dy)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_add_rms_norm_strides_zero_rows_and_the_sum_alone(dtype):
    g = gen(22)
    big = torch.randn(6, 50, 130, generator=g, device="cuda").to(dtype)
    w = torch.randn(64, generator=g, device="cuda").to(dtype)
    for x, r in ((big[..., :64], big[..., 64:128]), (big[..., 1:65], big[..., 3:67]),
                 (big.transpose(0, 1)[..., :64], big.transpose(0, 1)[..., :64]),
                 (big[:1, :, :64].expand(6, 50, 64), big[..., :128:2])):
        y, t = sequence.add_rms_norm(x, r, w)
        ry, rt = ref_norm(x, r, w)
        assert y.shape == x.shape
        assert err(y, ry) < NORM_TOL[dtype] and err(t, rt) < NORM_TOL[dtype]
    z = torch.zeros(3, 64, device="cuda", dtype=dtype, requires_grad=True)
    y, t = sequence.add_rms_norm(z, z, w)
    assert not y.any() and torch.isfinite(torch.autograd.grad(y, z, torch.ones_like(y))[0].float()).all()
    e = torch.zeros(0, 64, device="cuda", dtype=dtype, requires_grad=True)
    wl = w.clone().requires_grad_(True)
    y, t = sequence.add_rms_norm(e, e, wl)
    assert y.shape == (0, 64)
    assert not torch.autograd.grad(y, wl, torch.ones_like(y))[0].any()
    x = torch.randn(4, 64, generator=g, device="cuda").to(dtype).requires_grad_(True)
    y, t = sequence.add_rms_norm(x, x.detach(), w)
    ds = torch.randn(4, 64, generator=g, device="cuda").to(dtype)
    assert torch.equal(torch.autograd.grad(t, x, ds)[0], ds)


def test_add_rms_norm_gradient_against_differences():
    """Central differences along the gradient with steps of 2^-6 per element:
    (2^-6)^2 times third derivatives of order one."""
    g = gen(23)
    x, r, w = (torch.randn(*s, generator=g, device="cuda") for s in ((5, 40), (5, 40), (40,)))
    a, b = (torch.randn(5, 40, generator=g, device="cuda") for _ in range(2))

    def loss(xs):
        y, t = sequence.add_rms_norm(*xs)
        return (y.double() * a + t.double() * b).sum()

    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    got = torch.autograd.grad(sequence.add_rms_norm(*leaves), leaves, [a, b])
    for i, gi in enumerate(got):
        d = gi / gi.abs().max() * 2.0 ** -6
        with torch.no_grad():
            hi = loss([t + d if j == i else t for j, t in enumerate((x, r, w))])
            lo = loss([t - d if j == i else t for j, t in enumerate((x, r, w))])
        want = float((gi.double() * d).sum())
        assert abs(float(hi - lo) / 2 - want) < 5e-3 * abs(want)


# ---------------------------------------------------------------------------
# Gated linear layer
# ---------------------------------------------------------------------------
def ref_gated(x, wg, wu, act):
    g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    a = g * torch.sigmoid(g) if act == "silu" else 0.5 * g * (1 + torch.erf(g * 0.5 ** 0.5))
    return a * u


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d,f", [(1, 1, 1), (1, 16, 32), (3, 128, 341), (64, 128, 341), (65, 100, 130), (128, 64, 64),
                                      (129, 512, 257), (500, 7, 1000), (1000, 256, 30), (257, 1000, 70), (4097, 64, 96),
                                      (40000, 72, 136)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_linear(rows, d, f, act, dtype):
    g = gen(24)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, wg, wu = n(rows, d).to(dtype), (n(f, d) * d ** -0.5).to(dtype), (n(f, d) * d ** -0.5).to(dtype)
    dh = n(rows, f).to(dtype)
    want = ref_gated(x, wg, wu, act)
    plain = sequence.gated_linear(x, wg, wu, act)
    assert err(plain, want) < TOL[dtype]
    leaves = [t.requires_grad_(True) for t in (x, wg, wu)]
    h = sequence.gated_linear(x, wg, wu, act)
    assert torch.equal(h, plain)
    got = torch.autograd.grad(h, leaves, dh)
    refs = [t.detach().double().requires_grad_(True) for t in leaves]
    ref = torch.autograd.grad(ref_gated(*refs, act), refs, dh.double())
    for a, b, name in zip(got, ref, ("dx", "dw_gate", "dw_up")):
        assert a.dtype == dtype and err(a, b) < TOL[dtype], name
    again = torch.autograd.grad(sequence.gated_linear(x, wg, wu, act), leaves, dh)
    for a, b in zip(got, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_linear_partial_gradients_strides_and_empty(dtype):
    g = gen(25)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    x, wg, wu = n(2, 9, 80), n(48, 80), n(48, 80)
    dh = n(2, 9, 48)
    refs = [t.double().requires_grad_(True) for t in (x, wg, wu)]
    ref = torch.autograd.grad(ref_gated(*refs, "silu"), refs, dh.double())
    for i in range(3):
        xs = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, wg, wu))]
        got = torch.autograd.grad(sequence.gated_linear(*xs), xs[i], dh)[0]
        assert err(got, ref[i]) < TOL[dtype]
    big = n(2, 9, 200)
    for v in (big[..., 1:81], big[..., ::2][..., :80], big[:1, :, :80].expand(2, 9, 80)):
        h = sequence.gated_linear(v, wg, wu)
        assert h.shape == (2, 9, 48) and err(h, ref_gated(v, wg, wu, "silu")) < TOL[dtype]
    wt = n(80, 48).t()
    assert err(sequence.gated_linear(x, wt, wt), ref_gated(x, wt, wt, "silu")) < TOL[dtype]
    off = n(48 * 80 + 1)[1:].view(48, 80)
    assert err(sequence.gated_linear(x, off, off), ref_gated(x, off, off, "silu")) < TOL[dtype]
    e = torch.zeros(0, 80, device="cuda", dtype=dtype)
    wl = wg.clone().requires_grad_(True)
    h = sequence.gated_linear(e, wl, wu)
    assert h.shape == (0, 48)
    assert not torch.autograd.grad(h, wl, torch.ones_like(h))[0].any()


def test_gated_linear_saturated_activations():
    """exp(-g) overflows for large negative gates and the product with it stays 0, not NaN."""
    x = torch.tensor([[200.0], [-200.0], [30000.0], [-30000.0]], device="cuda", requires_grad=True)
    one = torch.ones(1, 1, device="cuda")
    for act in ("silu", "gelu"):
        h = sequence.gated_linear(x, one, one, act)
        want = torch.tensor([[4e4], [0.0], [9e8], [0.0]], device="cuda")
        assert torch.allclose(h, want, rtol=1e-5, atol=1e-30)
        dx = torch.autograd.grad(h, x, torch.ones_like(h))[0]
        assert torch.allclose(dx, torch.tensor([[400.0], [0.0], [6e4], [0.0]], device="cuda"), rtol=1e-5, atol=1e-30)


def test_gated_linear_gradient_against_differences():
    """Central differences along the gradient, steps of 2^-6 at most per element."""
    g = gen(26)
    x, wg, wu = torch.randn(20, 24, generator=g, device="cuda"), *(torch.randn(40, 24, generator=g, device="cuda") / 5
                                                                   for _ in range(2))
    a = torch.randn(20, 40, generator=g, device="cuda")
    for act in ("silu", "gelu"):
        leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
        got = torch.autograd.grad(sequence.gated_linear(*leaves, act), leaves, a)
        for i, gi in enumerate(got):
            d = gi / gi.abs().max() * 2.0 ** -6
            with torch.no_grad():
                hi, lo = ((sequence.gated_linear(*(t + s * d if j == i else t for j, t in enumerate((x, wg, wu))),
                                                 act).double() * a).sum() for s in (1, -1))
            want = float((gi.double() * d).sum())
            assert abs(float(hi - lo) / 2 - want) < 5e-3 * abs(want)


def test_operators_in_a_cuda_graph():
    """Captured and replayed on new inputs: nothing is kept from the capture."""
    q, k, v, g, S, _ = attention_inputs(8, 70, 4, 2, 64, 64, torch.bfloat16, 27)
    w = torch.randn(96, 64, generator=gen(28), device="cuda").bfloat16()
    one = torch.ones(64, device="cuda", dtype=torch.bfloat16)

    def step():
        o, st = sequence.linear_attention(q, k, v, g, initial_state=S, return_state=True)
        y, _ = sequence.add_rms_norm(o, q, one)
        return o, st, sequence.gated_linear(y, w, w), sequence.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, S)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    keep = S.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    q.copy_(torch.randn(q.shape, generator=gen(29), device="cuda"))
    S.copy_(keep)
    graph.replay()
    torch.cuda.synchronize()
    S.copy_(keep)
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# Sizes that select other kernels than the lists above
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows,d,f", [(20000, 264, 301), (12345, 512, 130), (19001, 256, 256)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_linear_pairs_of_blocks(rows, d, f, act):
    """Wide bfloat16 products over many tokens: two blocks share a tile; rows that
    end inside a pair's tile, odd row pitches, a reduction axis of one block and a half."""
    test_gated_linear(rows, d, f, act, torch.bfloat16)


@pytest.mark.parametrize("shape", [(3, 300, 2, 1, 128, 128), (2, 700, 4, 2, 72, 128), (2, 257, 2, 2, 128, 8),
                                   (1, 5000, 3, 3, 104, 96)], ids=str)
def test_wide_heads_ignore_what_lies_past_the_lengths(shape):
    """Heads of more than 64 elements, whole and in segments: NaN and infinities past
    the lengths reach nothing, gradients included."""
    q, k, v, g, S, L = attention_inputs(*shape, torch.bfloat16, 30, lengths="ragged")
    o, st = sequence.linear_attention(q, k, v, g, initial_state=S, lengths=L, return_state=True)
    ro, rs = ref_attention(q, k, v, g, S, L)
    assert err(o, ro) < TOL[torch.bfloat16] and err(st, rs) < F32_TOL
    dirty = [t.clone() for t in (q, k, v)]
    for t in dirty:
        for b in range(shape[0]):
            t[b, L[b]:] = float("nan") if b % 2 else float("inf")
    o2, st2 = sequence.linear_attention(*dirty, g, initial_state=S, lengths=L, return_state=True)
    assert torch.equal(o, o2) and torch.equal(st, st2)
    leaves, dleaves = ([t.clone().requires_grad_(True) for t in x] for x in ((q, k, v), dirty))
    do = torch.randn(o.shape, generator=gen(31), device="cuda").bfloat16()
    for a, b in zip(torch.autograd.grad(sequence.linear_attention(*leaves, g, lengths=L), leaves, do),
                    torch.autograd.grad(sequence.linear_attention(*dleaves, g, lengths=L), dleaves, do)):
        assert torch.equal(a, b)


def test_wide_heads_strided_broadcast_and_unaligned():
    """Views that the asynchronous copies can and cannot read."""
    B, T, H, D = 2, 200, 2, 128
    g = attention_inputs(B, T, H, H, D, D, torch.bfloat16, 0)[3]
    big = torch.randn(B, T, 3, H, D, generator=gen(32), device="cuda").bfloat16()
    odd = torch.randn(3, B * T * H * D + 1, generator=gen(33), device="cuda").bfloat16()
    for q, k, v in (tuple(big[:, :, i] for i in range(3)), tuple(odd[i, 1:].view(B, T, H, D) for i in range(3)),
                    tuple(big[:1, :, i].expand(B, T, H, D) for i in range(3)),
                    tuple(big[:, :1, i].expand(B, T, H, D) for i in range(3)),
                    tuple(big[..., :72][:, :, i] for i in range(3))):
        assert err(sequence.linear_attention(q, k, v, g), ref_attention(q, k, v, g)[0]) < TOL[torch.bfloat16]


def test_without_dlog_the_gradients_are_those_with_it():
    """log_decay without a gradient selects kernels with fewer terms: the results agree to bfloat16."""
    for D in (32, 64, 128):
        q, k, v, g, _, L = attention_inputs(3, 150, 4, 2, D, D, torch.bfloat16, 34, state=False, lengths="ragged")
        do = torch.randn(q.shape, generator=gen(35), device="cuda").bfloat16()
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        refs = [t.detach().double().requires_grad_(True) for t in leaves]
        want = torch.autograd.grad(ref_attention(*refs, g, None, L)[0], refs, do.double())
        for a, b in zip(torch.autograd.grad(sequence.linear_attention(*leaves, g, lengths=L), leaves, do), want):
            assert err(a, b) < TOL[torch.bfloat16]


def test_waits_that_run_out_leave_nan_and_a_usable_context():
    """With a poll limit of 0 every wait of the tensor-core kernels gives up at once (their
    copies do complete and are drained): the outputs are NaN, and the next call is right."""
    from turbompc_b200 import _ffi
    lib = _ffi.load()
    x = torch.randn(300, 128, generator=gen(36), device="cuda").bfloat16().requires_grad_(True)
    w = torch.randn(200, 128, generator=gen(37), device="cuda").bfloat16() / 11
    X = torch.randn(20000, 264, generator=gen(38), device="cuda").bfloat16()
    W = torch.randn(304, 264, generator=gen(39), device="cuda").bfloat16() / 16
    q, k, v, g, S, _ = attention_inputs(2, 300, 2, 1, 128, 128, torch.bfloat16, 40)
    before = lib.tmpc_set_transfer_poll_limit(0)
    try:
        h = sequence.gated_linear(x, w, w)
        dx, = torch.autograd.grad(h, x, torch.ones_like(h))
        H = sequence.gated_linear(X, W, W)
        o, st = sequence.linear_attention(q, k, v, g, initial_state=S, return_state=True)
        torch.cuda.synchronize()
    finally:
        lib.tmpc_set_transfer_poll_limit(before)
    assert torch.isnan(h).all() and torch.isnan(dx).all() and torch.isnan(H).all()
    assert torch.isnan(o).all() and torch.isnan(st).all()
    assert err(sequence.gated_linear(x, w, w).detach(), ref_gated(x.detach(), w, w, "silu")) < TOL[torch.bfloat16]
    assert err(sequence.gated_linear(X, W, W), ref_gated(X, W, W, "silu")) < TOL[torch.bfloat16]
    o, st = sequence.linear_attention(q, k, v, g, initial_state=S, return_state=True)
    ro, rs = ref_attention(q, k, v, g, S)
    assert err(o, ro) < TOL[torch.bfloat16] and err(st, rs) < F32_TOL


def test_gated_linear_from_a_thread_that_made_no_cuda_call():
    """The maps of the asynchronous copies are made by a driver call, which needs the
    device's context on the calling thread (a backward pass has a thread of its own)."""
    import threading
    x = torch.randn(300, 128, generator=gen(41), device="cuda").bfloat16()
    w = torch.randn(200, 128, generator=gen(42), device="cuda").bfloat16() / 11
    want = sequence.gated_linear(x, w, w)
    torch.empty(300, 200, device="cuda", dtype=torch.bfloat16)  # leaves a block for the thread's output
    got = []

    def work():
        with torch.no_grad():
            got.append(sequence.gated_linear(x, w, w))

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert len(got) == 1 and torch.equal(got[0], want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_linear_activation_in_its_tails(act, dtype):
    """One projection is g itself, the other 1: act(g) and act'(g) element by element, where act is tiny too.
    bfloat16: the result's rounding (2^-9) once, and less than that of the functions' errors; float: erfc's
    relative error per rounding of its argument, 2^-24 g^2 (81 at g = -9), twice, and some roundings."""
    g = torch.linspace(-9, 9, 3 * 128 + 5, device="cuda").to(dtype)
    x = torch.zeros(len(g), 16, device="cuda", dtype=dtype)
    x[:, 0], x[:, 1] = g, 1
    w = torch.zeros(2, 1, 16, device="cuda", dtype=dtype)
    w[0, 0, 0] = w[1, 0, 1] = 1
    x.requires_grad_(True)
    h = sequence.gated_linear(x, w[0], w[1], activation=act)
    dx, = torch.autograd.grad(h, x, torch.ones_like(h))
    r = g.double()
    if act == "silu":
        s = torch.sigmoid(r)
        a, parts = r * s, (s, r * s * (1 - s))
    else:
        c = 0.5 * torch.special.erfc(-r * 0.5 ** 0.5)
        a, parts = r * c, (c, r * torch.exp(-r * r / 2) * (2 * math.pi) ** -0.5)
    tol = 2.0 ** -8 if dtype == torch.bfloat16 else 200 * 2.0 ** -24
    assert float(((h.double()[:, 0] - a).abs() / a.abs().clamp(min=1e-30)).max()) < tol
    size = parts[0].abs() + parts[1].abs()
    assert float(((dx.double()[:, 0] - sum(parts)).abs() / size).max()) < tol
