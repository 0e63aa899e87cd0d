"""Multi-tensor Adam on the HIP kernel `clt_adam_step` -- the MI355X counterpart of the
``torch.optim.Adam(pgs, betas=(b1, b2))`` the reference builds in trainer.py:166-186
(eps 1e-8, no weight decay, no amsgrad; per-group lr, possibly a tensor; LambdaLR-compatible).

One launch updates every parameter of every group: the host refreshes a small table of
(p, g, m, v, numel, lr) records each step (grad pointers change when autograd allocates
new .grad tensors) and uploads it asynchronously; the chunk -> tensor map is static."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _lib
from .hip_ops import _DT, _call, _stream, adamw_step

import os

CHUNK = int(os.environ.get("CLT_ADAM_CHUNK", 1 << 14))  # elements per workgroup (a multiple of 8)


class Adam(torch.optim.Optimizer):
    HAS_STATE = True

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8):
        defaults = dict(lr=lr, betas=betas, eps=eps)
        super().__init__(params, defaults)
        self._step = 0
        self._tables = {}  # key: tuple of param ids with grads -> static device tables

    def state_dict(self):
        sd = super().state_dict()
        sd["clt_step"] = self._step  # one step count for all parameters (torch keeps one per parameter)
        return sd

    def load_state_dict(self, state_dict):
        sd = dict(state_dict)
        self._step = sd.pop("clt_step", self._step)
        super().load_state_dict(sd)
        self._tables = {}  # the cached pointer tables name the state tensors that were just replaced
        for cache in ("_group_of", "_by_ptr"):
            self.__dict__.pop(cache, None)

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for cache in ("_group_of", "_by_ptr"):
            self.__dict__.pop(cache, None)
        self._tables = {}

    def _state(self, p):
        st = self.state[p]
        if not st:
            st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
        return st

    def fused_rows(self, p):
        """State and hyper-parameters with which a gradient-producing kernel may apply THIS step's update of ``p``
        itself (hip_ops.spt_dense_adam); ``p`` must then reach step() without a .grad.  None if p is not ours."""
        if not hasattr(self, "_group_of"):
            self._group_of = {id(q): gi for gi, g in enumerate(self.param_groups) for q in g["params"]}
        gi = self._group_of.get(id(p))
        if gi is None:
            return None
        st = self._state(p)
        g = self.param_groups[gi]
        return dict(m=st["exp_avg"], v=st["exp_avg_sq"], lr=float(g["lr"]), betas=g["betas"], eps=g["eps"],
                    step=self._step + 1)

    def fused_rows_by_ptr(self, ptr: int):
        """fused_rows for the parameter whose storage starts at ``ptr`` (autograd Functions see saved tensors, not the
        Parameter objects).  Parameters that already hold a .grad are not eligible."""
        if not hasattr(self, "_by_ptr"):
            self._by_ptr = {q.data_ptr(): q for g in self.param_groups for q in g["params"]}
        p = self._by_ptr.get(ptr)
        if p is None or p.grad is not None:
            return None
        return self.fused_rows(p)

    @torch.no_grad()
    def step(self, closure=None):
        assert closure is None
        self._step += 1
        live = []
        for gi, group in enumerate(self.param_groups):
            for p in group["params"]:
                if p.grad is not None:
                    live.append((gi, p))
        if not live:
            return
        dev = live[0][1].device
        key = tuple(id(p) for _, p in live)
        tb = self._tables.get(key)
        if tb is None:
            ct, cs = [], []
            for ti, (_, p) in enumerate(live):
                n = p.numel()
                starts = np.arange(0, n, CHUNK, dtype=np.int64)
                ct.append(np.full(len(starts), ti, dtype=np.int32))
                cs.append(starts)
            ct = torch.from_numpy(np.concatenate(ct)).to(dev)
            cs = torch.from_numpy(np.concatenate(cs)).to(dev)
            # The upload below is asynchronous and the host may run several steps ahead of the GPU: a ring of pinned
            # staging buffers, each guarded by an event recorded after its copy, so that a buffer is never rewritten
            # (next step's lr, new .grad pointers) before the copy that reads it has executed.
            nbytes = len(live) * C.sizeof(_lib.AdamTensor)
            ring = [[torch.empty(nbytes, dtype=torch.uint8).pin_memory(), None] for _ in range(4)]
            devt = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            tb = self._tables[key] = (ct, cs, ring, devt)
        ct, cs, ring, devt = tb
        slot = ring[self._step % len(ring)]
        if slot[1] is not None:
            slot[1].synchronize()
        host = slot[0]
        recs = (_lib.AdamTensor * len(live)).from_address(host.data_ptr())
        for ti, (gi, p) in enumerate(live):
            g = p.grad
            if not g.is_contiguous():
                g = p.grad = g.contiguous()
            assert p.is_contiguous() and g.shape == p.shape
            r = recs[ti]
            if self.HAS_STATE:
                st = self._state(p)
                r.p, r.g, r.m, r.v = p.data_ptr(), g.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()
            else:
                r.p, r.g, r.m, r.v = p.data_ptr(), g.data_ptr(), None, None
            r.numel = p.numel()
            r.lr = float(self.param_groups[gi]["lr"])
            r.p_dtype, r.g_dtype = _DT[p.dtype], _DT[g.dtype]
        devt.copy_(host, non_blocking=True)
        slot[1] = torch.cuda.Event()
        slot[1].record()
        self._launch(devt, len(live), ct, cs)

    def _launch(self, devt, n_tensors, ct, cs):
        betas = self.param_groups[0]["betas"]
        eps = self.param_groups[0]["eps"]
        _call("clt_adam_step", C.c_void_p(devt.data_ptr()), n_tensors, C.c_void_p(ct.data_ptr()),
              C.c_void_p(cs.data_ptr()), ct.numel(), CHUNK, 1.0, float(betas[0]), float(betas[1]), float(eps),
              self._step, _stream(devt))


class SignSGD(Adam):
    """sparsify/sign_sgd.py:5-23 (steepest descent in the L-infinity norm): ``p -= lr * sign(p.grad)`` for every parameter
    that has a gradient, all tensors in one launch of ``clt_signsgd_step``.  No optimizer state."""

    HAS_STATE = False

    def __init__(self, params, lr: float = 1e-3):
        if lr <= 0.0:
            raise ValueError(f"Invalid learning rate: {lr}")
        torch.optim.Optimizer.__init__(self, params, {"lr": lr})
        self._step = 0
        self._tables = {}

    def fused_rows(self, p):  # no fused row-pass form: the gradient kernels write plain gradients for this optimizer
        return None

    def fused_rows_by_ptr(self, ptr):
        return None

    def _launch(self, devt, n_tensors, ct, cs):
        _call("clt_signsgd_step", C.c_void_p(devt.data_ptr()), n_tensors, C.c_void_p(ct.data_ptr()),
              C.c_void_p(cs.data_ptr()), ct.numel(), CHUNK, 1.0, _stream(devt))


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) on ``clt_adamw_step``: every parameter of a group in one call, with moments that do not
    take the parameter's type as ``Adam``'s do.  ``state_bits=32``: float32 moments, whatever the parameters are.
    ``state_bits=8``: one byte per element and moment (the first moment and the square root of the second in e4m3, one
    power of two for 128 elements, stochastic rounding: hip_ops.adamw_step) for every tensor of at least
    ``min_8bit_size`` elements; smaller ones keep float32 moments.  (The reference's optimizer with 8-bit moments:
    trainer.py:155-164.)  ``seed`` names the random bits: two runs with the same seed round alike.  Every parameter counts
    the steps that updated it, as ``torch.optim.AdamW``'s do: one whose first gradient comes late starts with step 1's bias
    correction.  Not capturable."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, *,
                 state_bits: int = 32, min_8bit_size: int = 4096, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is 8 or 32, got {state_bits}")
        if float(lr) < 0.0 or eps < 0.0 or weight_decay < 0.0 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"invalid hyper-parameters: lr {float(lr)}, betas {betas}, eps {eps}, weight_decay {weight_decay}")
        # (the last entry is for torch.optim.Adam, which goes on from a saved state by it)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, decoupled_weight_decay=True))
        self.state_bits, self.min_8bit_size, self.seed = state_bits, min_8bit_size, seed
        self._step = 0  # calls of step() that updated something
        self._steps = {}  # updates of each parameter

    def __getstate__(self):  # (of a copy or a pickle: torch's has the groups and the state alone)
        own = ("state_bits", "min_8bit_size", "seed", "_step", "_steps")
        return {**super().__getstate__(), **{name: getattr(self, name) for name in own}}

    def _moments(self, p):
        """The state of ``p`` as hip_ops.adamw_step takes it: (first, second)."""
        st = self.state[p]
        if not st:
            self._steps[p] = 0
        self._steps.setdefault(p, self._step)  # (a state put there from outside)
        if not st:
            if self.state_bits == 8 and p.numel() >= self.min_8bit_size:
                for name in ("exp_avg", "rms"):
                    st[name + "_codes"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
                    st[name + "_scales"] = torch.zeros(-(-p.numel() // 128), dtype=torch.uint8, device=p.device)
            else:
                st["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                st["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if "exp_avg" in st:
            return st["exp_avg"], st["exp_avg_sq"]
        return (st["exp_avg_codes"], st["exp_avg_scales"]), (st["rms_codes"], st["rms_scales"])

    @torch.no_grad()
    def step(self, closure=None):
        assert closure is None
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step cannot be captured into a graph: every replay would repeat the same step count")
        live = [(g, [p for p in g["params"] if p.grad is not None]) for g in self.param_groups]
        for _, ps in live:
            for p in ps:
                if p.grad.is_sparse or not p.is_contiguous():
                    raise RuntimeError("AdamW needs dense gradients and contiguous parameters")
        calls = {}  # what one call has in common -> its tensors; groups usually differ in lr alone, and counts are alike
        for group, ps in live:
            if ps:
                lr, wd = float(group["lr"]), float(group["weight_decay"])
                for p in ps:
                    m, v = self._moments(p)
                    key = (p.device, tuple(group["betas"]), group["eps"], self._steps[p] + 1)
                    c = calls.setdefault(key, ([], [], [], [], [], []))
                    for to, x in zip(c, (p, p.grad, m, v, lr, wd)):
                        to.append(x)
        for (_, betas, eps, step), (ps, gs, ms, vs, lrs, wds) in calls.items():
            adamw_step(ps, gs, ms, vs, step=step, lr=lrs, betas=betas, eps=eps, weight_decay=wds, seed=self.seed)
            for p in ps:  # (a call that was refused counts for nothing)
                self._steps[p] = step
        self._step += bool(calls)

    def state_dict(self):
        """As torch's (a parameter's count of updates is its state's ``step``), and ``clt_step``."""
        sd = super().state_dict()
        params = [p for g in self.param_groups for p in g["params"]]
        sd["state"] = {i: {**st, "step": torch.tensor(float(self._steps.get(params[i], self._step)))} if st else st for i, st in sd["state"].items()}
        sd["clt_step"] = self._step
        return sd

    def load_state_dict(self, state_dict):
        """Moments keep the type they were saved in (the base class would cast them to the parameter's)."""
        sd = dict(state_dict)
        saved = sd.get("state", {})
        for option in ("amsgrad", "maximize"):
            if any(g.get(option) for g in sd.get("param_groups", ())):
                raise ValueError(f"AdamW: the saved state was made with {option}=True")
        step = sd.pop("clt_step", None)
        counts = {i: int(st["step"]) for i, st in saved.items() if "step" in st}
        if step is None:  # (written by torch.optim)
            if len(set(counts.values())) > 1:
                raise ValueError("AdamW: one step count for all parameters is expected of a state without 'clt_step', the saved one has "
                                 f"{sorted(set(counts.values()))}; with state_dict['clt_step'] = {max(counts.values())} each keeps its own")
            step = max(counts.values(), default=self._step)
        params = [p for g in self.param_groups for p in g["params"]]
        state, steps = {}, {}
        for i, st in saved.items():
            p, n = params[i], params[i].numel()
            want = ({"exp_avg": (torch.float32, n), "exp_avg_sq": (torch.float32, n)} if "exp_avg" in st else
                    {name + part: (torch.uint8, size) for name in ("exp_avg", "rms")
                     for part, size in (("_codes", n), ("_scales", -(-n // 128)))})
            for name, (dtype, size) in want.items():
                if name not in st or st[name].numel() != size or (dtype == torch.uint8) != (st[name].dtype == torch.uint8):
                    raise ValueError(f"AdamW: the saved state of parameter {i} does not fit ({name})")
            steps[p] = counts.get(i, step)  # (what an earlier version saved has one count for all)
            state[p] = {name: st[name].detach().to(device=p.device, dtype=dtype, copy=True).contiguous()
                        for name, (dtype, _) in want.items()}
        super().load_state_dict({**sd, "state": {}})
        for g in self.param_groups:
            g["decoupled_weight_decay"] = True
        self.state.clear()
        self.state.update(state)
        self._step, self._steps = step, steps
