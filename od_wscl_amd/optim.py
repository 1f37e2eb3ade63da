"""AdamW over many tensors at once, and the global gradient norm it is clipped by (csrc/adamw.hip).

The reference trains with SGD only (solver/build.py:10-24, engine.FlatSGD here); this is the optimiser beside it, for heads
that do not train well under SGD.  Three ways in:

  * `ODW.OPTIMIZER "ADAMW"`: the training step of engine.build_training_step (tools/train_net.py) runs it over its flat buffers;
  * `AdamW`, a torch.optim.Optimizer, for a module of one's own;
  * `adamw_step` / `adamw8_step` / `grad_norm` / `clip_grad_norm_` on lists of tensors.

States are fp32, or 8-bit floats (2 bytes a parameter for both averages instead of 8): the first average in float8_e4m3fn,
the second in float8_e5m2, a power-of-two scale each for every 256 consecutive elements of a tensor, rounded stochastically with counter-based
bits (adamw8_step says which) -- a step is a function of its inputs and its key, whatever the launch geometry.

Every tensor is on one GPU; the work goes to the current stream of that device; nothing is read back to the host."""
import math
from collections import defaultdict

import torch

from . import _lib as L
from .utils import rng

BLOCK = 256          # elements that share a scale of the 8-bit states
STATE8 = {"exp_avg": torch.float8_e4m3fn, "exp_avg_sq": torch.float8_e5m2}
MIN_EPS = 1e-15      # (a smaller eps is refused: csrc/bind.cpp says why)


def _list(grads):
    return [grads] if torch.is_tensor(grads) else list(grads)          # (iterating over one parameter would give rows of its values)


def grad_norm(grads, max_norm=None):
    """The 2-norm over all of `grads` (tensors, or parameters that stand for their .grad; or one) as a 0-dim fp32 tensor; summed in fp64 in
    one order, so the same from run to run.  With max_norm: (norm, coef), coef = min(1, max_norm / (norm + 1e-6)) -- the factor
    that clips them, for `grad_scale` of adamw_step (clipping without a pass over the gradients).  Neither is read by the host.
    A non-finite gradient makes the norm inf or NaN, and coef 0 or NaN.  Not differentiable."""
    return L.bind().grad_norm(_list(grads), max_norm)


def clip_grad_norm_(grads, max_norm):
    """Scale all of `grads` (tensors, or parameters that stand for their .grad; or one; elements in any order without gaps) in place so that
    their common 2-norm is at most max_norm; returns the norm before that, 0 where none has a gradient (torch.nn.utils.clip_grad_norm_,
    without a host read)."""
    return L.bind().clip_grad_norm(_list(grads), max_norm)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, grad_scale=None,
               copies=None, grad_mult=1.0, max_workgroups=0):
    """One AdamW step over lists of tensors, in place, one launch for up to 48 of them:

        g' = g * grad_mult * grad_scale
        m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
        p -= lr (m / (1 - b1^step) / (sqrt(v / (1 - b2^step)) + eps) + weight_decay p)

    params fp32 or bf16 (updated in fp32, rounded once to nearest), grads fp32 or bf16, states fp32; all contiguous, none twice in a
    list, none overlapping.  lr, weight_decay: a number, or one per tensor.  step: the number of this step, from 1 -- or an int64
    tensor on the GPU that holds the steps taken and is advanced here, the form a HIP graph can capture.  grad_scale: one fp32 on the
    GPU (the clip coefficient of grad_norm).  copies: list of bf16 tensors (or None) that get the new params, as the matrix cores read
    them.  max_workgroups: 0, or the width of a pass that runs beside other work."""
    L.bind().adamw(False, params, grads, exp_avgs, exp_avg_sqs, None, step, (), lr, betas, eps, weight_decay, grad_scale, copies, grad_mult,
                   max_workgroups, True)


def adamw8_step(params, grads, exp_avgs, exp_avg_sqs, scales, step, key, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                grad_scale=None, copies=None, grad_mult=1.0, max_workgroups=0, hold_v=True):
    """adamw_step with 8-bit states: exp_avgs float8_e4m3fn, exp_avg_sqs float8_e5m2, scales uint8 (ceil(n / 256), 2): exponent + 127 of
    the power-of-two scales of the two averages of 256 elements; value = code * 2^(scale - 127) (state8_zeros, state8_read,
    state8_write).  The update uses the averages before they are rounded.  An average that is not finite is held as NaN.

    key: two 32-bit integers, other ones every step (utils.rng.stream_key(seed, step)).  The random bits of an element are mix(mix(i ^ k0)
    + k1) of utils/rng.py, i = its position in the concatenation of `params`, under the keys k0 = key[0] and k1 = key[1] + 0x9E3779B9 key[0]:
    keys that differ in the first word alone (a step's number, say) then do not permute one set of numbers over the elements.  With
    `step` on the GPU the step's number is added to k1.

    hold_v: a second average that is not zero is held as 2^-16 of its scale at least, which bounds the steps of elements far below their block's
    largest.  False: it is rounded to zero like any other value, and such an element may move by lr times its first average over eps."""
    L.bind().adamw(True, params, grads, exp_avgs, exp_avg_sqs, scales, step, key, lr, betas, eps, weight_decay, grad_scale, copies,
                   grad_mult, max_workgroups, hold_v)


# ---- the 8-bit states as tensors -----------------------------------------------------------------------------------------------------


def state8_zeros(p):
    """(exp_avg, exp_avg_sq, scales) of a parameter before its first step."""
    blocks = -(-p.numel() // BLOCK)
    return (torch.zeros(p.shape, dtype=torch.float8_e4m3fn, device=p.device), torch.zeros(p.shape, dtype=torch.float8_e5m2, device=p.device),
            torch.full((blocks, 2), 1, dtype=torch.uint8, device=p.device))


def state8_read(exp_avg, exp_avg_sq, scales):
    """The two averages as fp32 tensors: exactly what is held."""
    out = []
    for col, q in enumerate((exp_avg, exp_avg_sq)):
        s = (scales[:, col].to(torch.int32) << 23).view(torch.float32)          # (torch.ldexp goes through pow on the GPU: off by an ulp)
        out.append((q.reshape(-1).float() * s.repeat_interleave(BLOCK)[:q.numel()]).view(q.shape))
    return tuple(out)


def state8_write(m, v, out=None):
    """(exp_avg, exp_avg_sq, scales) that hold m and v, rounded to nearest; what state8_read gave comes back the same."""
    res = state8_zeros(m) if out is None else out
    for col, (x, q, top) in enumerate(((m, res[0], 8), (v, res[1], 15))):
        n = x.numel()
        blocks = torch.nn.functional.pad(x.detach().reshape(-1).float(), (0, -n % BLOCK)).view(-1, BLOCK)
        finite = torch.isfinite(blocks)
        a = torch.where(finite, blocks.abs(), torch.zeros_like(blocks)).amax(1)
        bits = a.view(torch.int32)
        e = ((bits >> 23) - top + ((bits & 0x7FFFFF) > 0x600000)).clamp(1, 254)
        y = torch.where(finite, blocks * ((254 - e) << 23).view(torch.float32).view(-1, 1), torch.full_like(blocks, math.nan))
        if col == 1:
            y = torch.where(blocks > 0, y.clamp_min(2.0 ** -16), y)
        q.copy_(y.view(-1)[:n].view(q.shape).to(q.dtype))
        res[2][:, col] = e.to(torch.uint8)
    return res


# ---- the optimiser object ------------------------------------------------------------------------------------------------------------


def refuse_other_rules(param_groups):
    """Groups of a torch optimiser whose averages mean, or whose steps did, something else than adamw_step's."""
    for g in param_groups:
        other = [k for k in ("amsgrad", "maximize") if g.get(k)] + ["coupled weight decay"] * (not g.get("decoupled_weight_decay", True))
        if other:
            raise ValueError("AdamW: the state is of an optimiser with %s" % ", ".join(other))


def _order(p):
    """The order of p's dimensions in memory where that is another one without gaps, else None."""
    if p.is_contiguous():
        return None
    order = sorted(range(p.dim()), key=lambda d: -p.stride(d))
    return order if p.permute(order).is_contiguous() else None


def _flat(t, order):
    """t's dimensions in that order: contiguous, if t lies like the parameter it is of."""
    return t if order is None else t.permute(order)


def _back(t, order):
    """What _flat undoes."""
    return t if order is None else t.permute([order.index(d) for d in range(len(order))])


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's arguments, groups and state names on the kernels above.  Parameters' elements may lie in any order without gaps
    (channels_last weights); the averages lie like them.

    state_bits: 32, or 8.  max_grad_norm: clip the gradients' common 2-norm (over all groups) within the step.  seed: of the 8-bit
    states' rounding.  capturable: the step's number lives on the GPU, so that step() can be captured into a HIP graph (learning
    rates are then those of the capture).  A captured step's parameters keep their step numbers together: an eager step of other betas or
    with a gradient missing gives some of them numbers of their own, and the step has to be captured again.

    state_dict() holds the averages in fp32 whatever state_bits is (an 8-bit state is read exactly and comes back the same), so
    checkpoints move between 32 and 8 bits and torch.optim.AdamW."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_grad_norm=None, seed=0,
                 capturable=False):
        if state_bits not in (8, 32):
            raise ValueError("AdamW: state_bits = %r (8 | 32)" % (state_bits,))
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError("AdamW: max_grad_norm = %r" % (max_grad_norm,))
        for name, x in (("lr", lr), ("weight_decay", weight_decay)):
            if not (x >= 0.0 and math.isfinite(x)):
                raise ValueError("AdamW: %s = %r" % (name, x))
        if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("AdamW: betas = %r" % (betas,))
        if not (eps >= MIN_EPS and math.isfinite(eps)):
            raise ValueError("AdamW: eps = %r" % (eps,))
        self.state_bits, self.max_grad_norm, self.seed, self.capturable = state_bits, max_grad_norm, int(seed), bool(capturable)
        self.grad_norm = None            # of the last step, where it was clipped (0-dim, on the GPU)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    # Copies and pickles: the base class keeps its own attributes only, and a plain pickle knows no 8-bit floats (they go as bytes).
    def __getstate__(self):
        own = ("state_bits", "max_grad_norm", "seed", "capturable", "grad_norm")
        data = dict(super().__getstate__(), **{k: self.__dict__[k] for k in own})
        if self.state_bits == 8:
            data["state"] = defaultdict(dict, {p: dict(st, **{k: st[k].view(torch.uint8) for k in STATE8}) for p, st in self.state.items()})
        return data

    def __setstate__(self, data):
        super().__setstate__(data)
        if self.state_bits == 8:
            for st in self.state.values():
                st.update({k: st[k].view(t) for k, t in STATE8.items()})

    def _state(self, p, order):
        st = self.state[p]
        if not st:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                del self.state[p]
                raise RuntimeError("AdamW: a parameter's first step is being captured: every replay would start it from zero averages again "
                                   "(take a step, or load a state, before the capture)")
            self._hold(st, p, order)
            st["step"] = None            # (set by step(): a number, or with `capturable` a tensor that parameters share)
        elif not _flat(st["exp_avg"], order).is_contiguous():               # (the parameter was laid out anew)
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: a parameter's elements lie in another order than in the last step; take a step before the capture")
            self._hold(st, p, order, *self._averages(st))
        return st

    def _hold(self, st, p, order, m=None, v=None):
        """The averages m and v (fp32; none: zeros) in p's order, as they are held."""
        flat = _flat(p, order)
        if self.state_bits == 8:
            state = state8_zeros(flat) if m is None else state8_write(*(_flat(x, order).contiguous() for x in (m, v)))
            st["scales"] = state[2]
        else:
            state = [torch.zeros_like(flat, dtype=torch.float32, memory_format=torch.contiguous_format) for _ in range(2)]
            for x, given in zip(state, (m, v)):
                if given is not None:
                    x.copy_(_flat(given, order))
        st["exp_avg"], st["exp_avg_sq"] = (_back(x, order) for x in state[:2])

    @staticmethod
    def _averages(st):
        """Both averages in fp32: of an 8-bit state what it holds."""
        if "scales" not in st:
            return st["exp_avg"], st["exp_avg_sq"]
        order = _order(st["exp_avg"])
        return tuple(_back(x, order) for x in state8_read(*(_flat(st[k], order) for k in STATE8), st["scales"]))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls, grads, fresh = {}, [], {}          # (fresh: the counters made in this step)
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise TypeError("AdamW: sparse gradient")
                order = _order(p)
                st = self._state(p, order)
                rule = (tuple(group["betas"]), group["eps"])
                if st["step"] is None:
                    st["step"] = self._counter(fresh, (p.device,) + rule, 0, p.device) if self.capturable else 0
                # (a gradient that requires grad would stand for its own in grad_norm)
                g = p.grad.detach() if p.grad.requires_grad else p.grad
                g = _flat(g.resolve_neg(), order).contiguous()
                grads.append(g)
                number = id(st["step"]) if self.capturable else st["step"]
                calls.setdefault(rule + (number,), []).append((group, p, g, st, order))
        if not grads:
            return loss
        coef = None
        if self.max_grad_norm is not None:
            self.grad_norm, coef = grad_norm(grads, self.max_grad_norm)
        if self.capturable:
            self._part_counters(calls)
        for ci, ((betas, eps, _), items) in enumerate(calls.items()):
            step = items[0][3]["step"]
            if not self.capturable:
                step += 1
            ps, gs = [_flat(x[1], x[4]) for x in items], [x[2] for x in items]
            m, v = ([_flat(x[3][k], x[4]) for x in items] for k in ("exp_avg", "exp_avg_sq"))
            lr, wd = ([x[0][k] for x in items] for k in ("lr", "weight_decay"))
            more = dict(lr=lr, weight_decay=wd, betas=betas, eps=eps, grad_scale=coef)
            if self.state_bits == 8:
                # (a step whose number is on the GPU adds it to the key there)
                key = rng.stream_key(self.seed, (ci << 40) + (0 if self.capturable else step))
                adamw8_step(ps, gs, m, v, [x[3]["scales"] for x in items], step, key, **more)
            else:
                adamw_step(ps, gs, m, v, step, **more)
            if not self.capturable:
                for x in items:
                    x[3]["step"] = step
        return loss

    @staticmethod
    def _counter(made, key, value, device):
        if key not in made:
            made[key] = torch.full((1,), value, dtype=torch.int64, device=device)
        return made[key]

    def _part_counters(self, calls):
        """Parameters that took their first step together, by one rule, share a counter on the GPU: a step advances it once, for all of them.
        Those that part -- by a group's new betas or eps, or because only some have a gradient -- get counters of their own here; a step that
        is being captured cannot do that (its replays would take the copies' values anew)."""
        stepped = set(id(x[1]) for items in calls.values() for x in items)
        taken, apart = set(), {}
        for items in calls.values():
            counter = items[0][3]["step"]
            if id(counter) in taken:             # (another rule's call has it)
                apart[id(items[0][1])] = counter, [x[3] for x in items]
            taken.add(id(counter))
        for p, st in self.state.items():
            if id(st.get("step")) in taken and id(p) not in stepped:
                apart.setdefault(("rest", id(st["step"])), (st["step"], []))[1].append(st)
        if apart and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: parameters that share a step counter part in a captured step (other betas or eps, or a missing "
                               "gradient): take such a step before the capture")
        for counter, states in apart.values():
            own = counter.clone()
            for st in states:
                st["step"] = own

    def state_dict(self):
        """torch.optim.AdamW's layout: {"step": fp32 tensor, "exp_avg", "exp_avg_sq": fp32} a parameter."""
        sd = super().state_dict()
        for i, st in sd["state"].items():
            m, v = self._averages(st)
            sd["state"][i] = {"step": torch.tensor(float(st["step"])), "exp_avg": m, "exp_avg_sq": v}
        return sd

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """A state_dict() of this class (of either state_bits) or of torch.optim.AdamW (without amsgrad and maximize)."""
        refuse_other_rules(state_dict["param_groups"])
        states = dict(state_dict["state"])
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        shared = {}
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        own = [p for g in self.param_groups for p in g["params"]]
        rules = {id(p): (tuple(g["betas"]), g["eps"]) for g in self.param_groups for p in g["params"]}
        for i, p in zip(saved, own):
            if i not in states:
                continue
            step = int(states[i]["step"])
            st = self.state[p]
            m, v = (states[i][k].detach().to(device=p.device, dtype=torch.float32).reshape(p.shape) for k in ("exp_avg", "exp_avg_sq"))
            self._hold(st, p, _order(p), m, v)
            st["step"] = step
            if self.capturable:
                rule = rules[id(p)]
                st["step"] = self._counter(shared, (p.device, step) + rule, step, p.device)
