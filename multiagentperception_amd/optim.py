"""Optimizers on the HIP kernels (ops.adamw_step): what ``train_ops.GraphedTrainStep`` and ``parallel.agent_parallel_train_step`` take as
``optimizer``.  A step is a few launches for all tensors, reads nothing back to the host and keeps its counters on the device, so it is captured
as it is."""
import torch

from . import ops


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over f32, bf16 and f16 parameters on the GPU; half parameters are updated in f32 and rounded once, to
    nearest -- keep f32 parameters where an update is smaller than half a step of the type.

    state_bits 32: f32 moments; 8: moments in 8 bits (ops.adamw_step: e4m3 with a power-of-two scale per 256 elements, rounded at random by
    `seed`), 2 bytes an element in place of 8.  max_norm: all groups' gradients together are scaled down to this norm; `last_norm` is the
    norm before that (f32 on the device).  lr: a number (a schedule may change it between eager steps) or an f32 device tensor of one
    element, which captured steps follow.  A parameter without a gradient is left out of the step.  eps may be 0: an element that has had no
    gradient (none whose square f32 holds) is then only decayed."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_norm=None, seed=0):
        if state_bits not in (8, 32):
            raise ValueError("AdamW: state_bits is 8 or 32, got %r" % (state_bits,))
        if not torch.is_tensor(lr) and not lr >= 0.0:
            raise ValueError("AdamW: lr must not be negative, got %r" % (lr,))
        if not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0 or not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError("AdamW: betas in [0, 1), eps and weight_decay not negative, got %r, %r, %r" % (betas, eps, weight_decay))
        if max_norm is not None and not max_norm > 0.0:
            raise ValueError("AdamW: max_norm must be positive, got %r" % (max_norm,))
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=seed))
        self.max_norm, self.last_norm = max_norm, None

    @staticmethod
    def _fresh(p, bits):
        state = {"step": torch.zeros((), dtype=torch.float32, device=p.device)}
        if bits == 32:
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
            return state
        n, blocks = p.numel(), -(-p.numel() // ops.ADAMW_STATE_BLOCK)
        for name in ("exp_avg", "exp_avg_sq_root"):
            state[name] = torch.zeros(n, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
            state[name + "_scale"] = torch.zeros(blocks, dtype=torch.uint8, device=p.device).view(torch.float8_e8m0fnu)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = []
        for group in self.param_groups:
            params, grads, states, steps = [], [], [], []
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.layout != torch.strided:
                    raise ops.W2CError("AdamW: sparse gradients are not supported")
                if g.stride() != p.stride() and not (p.is_contiguous() and g.is_contiguous()):
                    g = torch.empty_like(p).copy_(g)                 # autograd laid it out otherwise than the parameter
                s = self.state[p]
                if not s:
                    s.update(self._fresh(p, group["state_bits"]))
                params.append(p)
                grads.append(g)
                steps.append(s["step"])
                if group["state_bits"] == 32:
                    states.append((s["exp_avg"], s["exp_avg_sq"]))
                else:
                    states.append((s["exp_avg"], s["exp_avg_scale"], s["exp_avg_sq_root"], s["exp_avg_sq_root_scale"]))
            if params:
                work.append((group, params, grads, states, steps))
        squares = None
        if self.max_norm is not None and work:
            squares = ops.grad_squares([g for _, _, grads, _, _ in work for g in grads])
        for group, params, grads, states, steps in work:
            norm = ops.adamw_step(params, grads, states, steps, group["lr"], group["betas"][0], group["betas"][1], group["eps"],
                                  group["weight_decay"], max_norm=self.max_norm, seed=group["seed"], squares=squares)
            if norm is not None:
                self.last_norm = norm
        return loss

    def load_state_dict(self, state_dict):
        """as torch's, but the moments and steps keep the types they were saved with (the base class casts them to the parameters')"""
        super().load_state_dict(state_dict)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            for k, v in state_dict["state"].get(i, {}).items():
                self.state[p][k] = v.detach().to(device=p.device, copy=True) if torch.is_tensor(v) else v
