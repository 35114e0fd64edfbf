"""A learned estimator in front of the MPC solve, trained through it.

Task: a spacecraft (Clohessy-Wiltshire relative motion) has to hold at a point
that it only knows from noisy measurements, one per control tick; the point
differs per environment.  ``HistoryEncoder`` reads an environment's history of
(measured point, state, control) tokens and emits the point; the MPC problem
takes it as its reference.  The encoder is trained by imitation: the loss is the
squared difference between the first control of its solve and that of an expert
who knows the point, and its gradient reaches the encoder's weights through the
solver's VJP.  In the closed loop the encoder runs one token per tick.

    python -m turbompc_b200.history_policy [--steps 200] [--batch 256]
        [--history 60] [--ticks 40] [--dtype float32|bfloat16] [--out results.json]
"""
from __future__ import annotations

import argparse
import json
from typing import Dict, Tuple

import numpy as np
import torch

from .dynamics import LinearDynamics
from .dynamics.integrators import predict_next_state
from .encoder import HistoryEncoder, last_outputs
from .problems.learned_cost import cw_matrices
from .problems.ocp import OptimalControlProblem
from .solver import TurboMPCSolver

NX, NU = 6, 3
REFERENCE = "reference_state_trajectory"


def make_problem(batch: int, horizon: int, dt: float, u_max: float, dtype, device):
    """Clohessy-Wiltshire tracking problem with a reference per environment."""
    A, B = cw_matrices()
    t = lambda a: torch.as_tensor(np.array(a), dtype=dtype, device=device)
    params = {
        "horizon": horizon, "discretization_resolution": dt, "discretization_scheme": 2,
        "initial_state": torch.zeros(batch, NX, dtype=dtype, device=device),
        "initial_guess_final_state": t(np.zeros(NX)),
        REFERENCE: torch.zeros(batch, horizon + 1, NX, dtype=dtype, device=device),
        "reference_control_trajectory": t(np.zeros(NU)), "penalize_control_reference": False,
        "weights_penalization_reference_state_trajectory": t(np.array([1.0] * 3 + [0.5] * 3)),
        "weights_penalization_final_state": t(np.full(NX, 5.0)),
        "weights_penalization_control_squared": t(np.full(NU, 0.5)),
        "weights_penalization_control_rate": t(np.zeros(NU)),
        "state_min_bounds": t(np.full(NX, -1e9)), "state_max_bounds": t(np.full(NX, 1e9)),
        "control_min_bounds": t(np.full(NU, -u_max)), "control_max_bounds": t(np.full(NU, u_max)),
        "dynamics_state_dot_params": {"A": t(A), "B": t(B)},
    }
    return OptimalControlProblem(LinearDynamics(NX, NU), params), params


class Experiment:
    """The environments, the solver around them, and the encoder."""

    def __init__(self, batch: int = 256, history: int = 60, horizon: int = 10, dt: float = 0.5, u_max: float = 2.0,
                 noise: float = 1.0, seed: int = 0, dtype=torch.float32, device="cuda"):
        self.batch, self.history, self.horizon, self.dt, self.noise = batch, history, horizon, dt, noise
        self.u_max, self.dtype, self.device = u_max, dtype, device
        self.program, self.params = make_problem(batch, horizon, dt, u_max, torch.float32, device)
        config = {"num_sqp_iteration_max": 1, "tol_convergence": 0.0,
                  "admm": {"max_iter": 100, "check_termination_every": 0, "adapt_rho_every": 0, "eps_abs": 1e-6,
                           "eps_rel": 1e-6, "pcg": {"max_iter": 30, "tol_epsilon": 0.0}}}
        self.solver = TurboMPCSolver(self.program, config, forward_backend="b200_direct", backward_backend="b200")
        torch.manual_seed(seed)
        self.encoder = HistoryEncoder(3 + NX + NU, 3, d_model=64, heads=4, kv_heads=2, head_dim=32, layers=2,
                                      dtype=dtype, device=device)
        self.gen = torch.Generator(device=device).manual_seed(seed + 1)
        self.dyn = self.program._dyn_params(self.params, self.params["initial_state"])

    def normal(self, *shape) -> torch.Tensor:
        return torch.randn(*shape, generator=self.gen, device=self.device)

    def advance(self, x: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
        return predict_next_state(self.program.dynamics, self.dt, 2, self.dyn, x, u)

    def token(self, x, u, point) -> torch.Tensor:
        measured = point + self.noise * self.normal(self.batch, 3)
        return torch.cat([measured, x, u], 1).to(self.dtype)

    @torch.no_grad()
    def histories(self) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """(points, tokens, lengths, final states): random controls, different lengths."""
        point, x = self.normal(self.batch, 3), torch.cat([self.normal(self.batch, 3), 0.1 * self.normal(self.batch, 3)], 1)
        lengths = torch.randint(1, self.history + 1, (self.batch,), generator=self.gen, device=self.device,
                                dtype=torch.int32)
        tokens, final = [], x
        for t in range(self.history):
            u = 0.05 * self.normal(self.batch, NU)
            tokens.append(self.token(x, u, point))
            final = torch.where((lengths == t + 1)[:, None], x, final)
            x = self.advance(x, u)
        return point, torch.stack(tokens, 1), lengths, final

    def first_control(self, x: torch.Tensor, point: torch.Tensor) -> torch.Tensor:
        """The solve's first control towards ``point`` from ``x``; differentiable in both."""
        reference = torch.cat([point, torch.zeros_like(point)], 1)[:, None].expand(-1, self.horizon + 1, -1)
        params = dict(self.params, initial_state=x.detach())
        solution = self.solver.solve(self.solver.initial_guess(params), params,
                                     {"initial_state": x, REFERENCE: reference})
        return solution.controls[:, 0]

    def estimate(self, tokens, lengths) -> torch.Tensor:
        outputs, _ = self.encoder(tokens, lengths)
        return last_outputs(outputs, lengths).float()

    def train(self, steps: int, lr: float = 3e-3, log=None) -> Dict[str, float]:
        opt = torch.optim.AdamW(self.encoder.parameters(), lr=lr, weight_decay=1e-4)
        losses = []
        for i in range(steps):
            for group in opt.param_groups:
                group["lr"] = lr * 0.5 * (1 + np.cos(np.pi * i / max(steps, 1)))
            point, tokens, lengths, final = self.histories()
            with torch.no_grad():
                expert = self.first_control(final, point)
            loss = (self.first_control(final, self.estimate(tokens, lengths)) - expert).pow(2).mean()
            opt.zero_grad(set_to_none=True)
            loss.backward()
            opt.step()
            losses.append(float(loss.detach()))
            if log and (i % 20 == 0 or i + 1 == steps):
                log(f"step {i:4d}  control error {losses[-1] ** 0.5:.4f}")
        return {"first_loss": float(np.mean(losses[:5])), "last_loss": float(np.mean(losses[-5:]))}

    @torch.no_grad()
    def closed_loop(self, ticks: int) -> Dict[str, float]:
        """One token per tick and environment: mean distance to the point at the
        end, with the encoder's estimates and with the last measurement alone."""
        out = {}
        for name in ("encoder", "measurement"):
            self.gen.manual_seed(1234)
            point = self.normal(self.batch, 3)
            x = torch.cat([3 * self.normal(self.batch, 3), torch.zeros(self.batch, 3, device=self.device)], 1)
            u = torch.zeros(self.batch, NU, device=self.device)
            state = self.encoder.initial_state(self.batch)
            dist = []
            for _ in range(ticks):
                token = self.token(x, u, point)
                estimate = self.encoder.step(token, state) if name == "encoder" else token[:, :3]
                u = self.first_control(x, estimate.float())
                x = self.advance(x, u)
                dist.append((x[:, :3] - point).norm(dim=1).mean())
            out[f"{name}_distance"] = float(torch.stack(dist[-10:]).mean())
        return out


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch", type=int, default=256)
    ap.add_argument("--history", type=int, default=60)
    ap.add_argument("--ticks", type=int, default=40)
    ap.add_argument("--dtype", choices=("float32", "bfloat16"), default="float32")
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--out", default="", help="write the results as JSON")
    args = ap.parse_args(argv)
    e = Experiment(batch=args.batch, history=args.history, seed=args.seed, dtype=getattr(torch, args.dtype))
    res = e.train(args.steps, log=lambda s: print(s, flush=True))
    res.update(e.closed_loop(args.ticks))
    print(json.dumps({"history_policy": res, "config": vars(args)}))
    if args.out:
        with open(args.out, "w") as f:
            json.dump({"history_policy": res, "config": vars(args)}, f, indent=1)
    return res


if __name__ == "__main__":
    main()
