"""The history encoder and the policy trained through the solve."""
import pytest
import torch
import torch.nn.functional as F

from turbompc_b200.encoder import HistoryEncoder, last_outputs
from turbompc_b200.history_policy import Experiment

pytestmark = pytest.mark.gpu


def _reference(enc, tokens):
    """The same model in plain 64-bit operations."""
    w = lambda p: p.detach().double()
    norm = lambda t, g: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * w(g)
    x, r = F.linear(tokens.double(), w(enc.w_in)), 0
    for l in enc.layers:
        r = x + r
        H, G, D = l.heads, l.kv_heads, l.head_dim
        p = F.linear(norm(r, l.norm_attention), w(l.w_qkv)).unflatten(-1, (H + 2 * G, D))
        q, k, v = p[..., :H, :], p[..., H:H + G, :].repeat_interleave(H // G, -2), p[..., H + G:, :].repeat_interleave(
            H // G, -2)
        d = torch.exp(w(l.log_decay()))[None, :, None, None]
        S, out = 0, []
        for t in range(tokens.shape[1]):
            S = d * S + k[:, t, :, :, None] * v[:, t, :, None, :]
            out.append(D ** -0.5 * (q[:, t, :, :, None] * S).sum(2))
        r = F.linear(torch.stack(out, 1).flatten(-2), w(l.w_out)) + r
        y = norm(r, l.norm_gated)
        x = F.linear(F.silu(F.linear(y, w(l.w_gate))) * F.linear(y, w(l.w_up)), w(l.w_down))
    return F.linear(norm(x + r, enc.norm_out), w(enc.w_out), w(enc.b_out))


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2.0 ** -13), (torch.bfloat16, 2.0 ** -4)])
def test_encoder_matches_plain_model_and_steps_match_sequences(dtype, tol):
    """Tolerances: two layers of operators at 2^-15 (float32) or a few 2^-9
    (bfloat16) each and as many library products, errors adding up."""
    torch.manual_seed(0)
    enc = HistoryEncoder(12, 5, d_model=64, heads=4, kv_heads=2, head_dim=32, hidden=170, dtype=dtype)
    tokens = torch.randn(7, 90, 12, device="cuda").to(dtype)
    want = _reference(enc, tokens)
    with torch.no_grad():
        got, end = enc(tokens)
        assert float((got.double() - want).norm() / want.norm()) < tol
        head, state = enc(tokens[:, :80])
        for t in range(80, 90):
            y = enc.step(tokens[:, t], state)
            assert float((y.double() - want[:, t]).norm() / want[:, t].norm()) < tol
        for a, b in zip(state, end):
            assert float((a - b).norm() / b.norm()) < tol
        # a shorter history gives what the whole one gives at its last token
        lengths = torch.tensor([90, 1, 40, 89, 64, 65, 7], dtype=torch.int32, device="cuda")
        y, _ = enc(tokens, lengths)
        last = want.gather(1, (lengths.long() - 1)[:, None, None].expand(-1, 1, 5))[:, 0]
        assert float((last_outputs(y, lengths).double() - last).norm() / last.norm()) < tol


def test_encoder_gradients_reach_every_parameter():
    enc = HistoryEncoder(12, 3, d_model=64, heads=4, kv_heads=2, head_dim=16)
    y, state = enc(torch.randn(3, 70, 12, device="cuda"))
    (y.square().sum() + sum(s.square().sum() for s in state)).backward()
    for name, p in enc.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, name


def test_encoder_refusals():
    with pytest.raises(ValueError):
        HistoryEncoder(4, 2, heads=4, kv_heads=3)
    enc = HistoryEncoder(4, 2, d_model=32, heads=2, head_dim=16)
    with pytest.raises(ValueError):
        enc(torch.zeros(2, 3, 5, device="cuda"))
    with pytest.raises(ValueError):
        enc.step(torch.zeros(2, 3, 4, device="cuda"), enc.initial_state(2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_policy_learns_through_the_solve(dtype):
    e = Experiment(batch=64, history=40, seed=3, dtype=dtype)
    res = e.train(60)
    assert res["last_loss"] < 0.5 * res["first_loss"], res
    loop = e.closed_loop(25)
    assert loop["encoder_distance"] < loop["measurement_distance"], loop
