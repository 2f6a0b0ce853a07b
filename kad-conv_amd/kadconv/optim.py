"""AdamW over a network's tensors in one launch (kad_adamw_step).

* ``AdamWPlan`` -- the step for tensors whose parameters and gradients stay where
  they are: a table of them is laid out on the GPU once.
* ``AdamW`` -- a ``torch.optim.Optimizer`` on such plans, which lays a table out
  anew when gradients have moved.

A detector has thousands of parameter tensors, half of them smaller than a
wave's load (KAD-CNet-S: 2944, median 22 values), so a step a tensor is bound by
its launches.

States are kept for all tensors of a plan in flat buffers, in the order of each
parameter's memory, each tensor's part beginning at a multiple of 256 values:

  32 bits   exp_avg, exp_avg_sq                    float32
  8 bits    exp_avg, exp_avg_sq_root               float8_e4m3fn, the numbers held
            exp_avg_scale, exp_avg_sq_root_scale   float32, one for 256 of them
  either    master                                 float32, with master_weights

8-bit states hold m and sqrt(v) as e4m3 numbers times their segment's scale
(its largest magnitude / 448), rounded stochastically with bits that are a hash
of (seed, step, place): the same call gives the same result.  A segment that
meets an infinity or NaN holds NaN from then on, as a single value does in 32 bits.
"""
import functools
import operator

import torch

from . import _ext

_NAMES = {32: ('exp_avg', 'exp_avg_sq'),
          8: ('exp_avg', 'exp_avg_sq_root', 'exp_avg_scale', 'exp_avg_sq_root_scale')}

# Of a parameter group; torch's base class adds its own.
_OPTIONS = {'lr', 'betas', 'eps', 'weight_decay', 'state_bits', 'master_weights', 'seed', 'capturable', 'step'}


def _same_layout(a, b):
    return a.shape == b.shape and (a.stride() == b.stride() or all(
        sa == sb for sa, sb, n in zip(a.stride(), b.stride(), a.shape) if n != 1))


def _check_rates(lr, betas, eps, weight_decay):
    if not isinstance(lr, torch.Tensor) and not lr >= 0:
        raise ValueError(f'lr must be >= 0, got {lr}')
    if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
        raise ValueError(f'betas must lie in [0, 1), got {betas}')
    if not (eps >= 0 and weight_decay >= 0):
        raise ValueError(f'eps and weight_decay must be >= 0, got {eps} and {weight_decay}')


class AdamWPlan:
    """The AdamW step of ``params`` by ``grads``, two lists of dense GPU tensors of one dtype (fp32, fp16 or
    bf16), equal in shapes and strides.  The plan holds their addresses: it is for tensors that keep their
    memory from step to step, as persistent gradient buffers and captured graphs do; ``set_grads`` takes
    others.  A gradient may be None: its parameter has a place in the state but is not stepped.

    ``state_bits`` 32 or 8; ``master_weights`` (16-bit parameters): an fp32 copy of them is stepped and rounded to
    them; ``state``: a dict of flat state buffers to use as they are, in place of new ones of zeros (and
    masters copied from the parameters); ``seed``: of the 8-bit states' stochastic rounding.

    With masters, values of a parameter that were written since its last step (a state dict loaded, an average swapped
    in, a clamp) take over from theirs.  A write that its version does not tell, through ``.data`` or to an inference
    tensor, is taken up by captured steps alone.

    ``plan.state`` holds the buffers."""

    def __init__(self, params, grads, state_bits=32, master_weights=False, state=None, seed=0):
        params = list(params)
        if state_bits not in _NAMES:
            raise ValueError(f'state_bits must be 32 or 8, got {state_bits}')
        self._table = _ext.native().AdamWTable(params)
        p0 = params[0]
        if master_weights and p0.dtype == torch.float32:
            raise ValueError('master weights are for 16-bit parameters')
        self.state_bits, self.master_weights, self.seed = state_bits, bool(master_weights), int(seed) & 0xFFFFFFFF
        self.device, self.state_elems = p0.device, self._table.elems
        self.set_grads(grads)
        self.state = self._new_state() if state is None else self._given_state(state)
        self._hand_over()

    def _hand_over(self):
        self._table.set_state(*(self.state[n] for n in _NAMES[self.state_bits]), *(None, None) * (self.state_bits == 32),
                              self.state.get('master'), self.state_bits, self.seed)

    def _reseed(self, seed):
        if self.seed != int(seed) & 0xFFFFFFFF:
            self.seed = int(seed) & 0xFFFFFFFF
            self._hand_over()

    @functools.cached_property
    def params(self):
        """The parameters, detached."""
        return self._table.params

    @functools.cached_property
    def offsets(self):
        """Where each parameter's part of a state buffer begins."""
        return self._table.offsets

    @functools.cached_property
    def _numels(self):
        return self._table.numels

    def _layout(self):
        """{name: (values, dtype)} of the state buffers."""
        n, seg = self.state_elems, _ext.ADAMW_SEG
        out = {}
        for name in _NAMES[self.state_bits]:
            if name.endswith('_scale'):
                out[name] = n // seg, torch.float32
            else:
                out[name] = n, torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn
        if self.master_weights:
            out['master'] = n, torch.float32
        return out

    def _new_state(self):
        state = {}
        for name, (n, dtype) in self._layout().items():
            state[name] = torch.zeros(n, dtype=torch.uint8 if dtype == torch.float8_e4m3fn else dtype,
                                      device=self.device).view(dtype)
        self._copy_masters(state)
        return state

    def _copy_masters(self, state):
        if self.master_weights:
            for i, p in enumerate(self.params):
                self.part(state['master'], i).copy_(p)

    def _start_over(self):
        """The state of a plan that has not stepped, in the same buffers."""
        for name, t in self.state.items():
            if name != 'master':
                t.view(torch.uint8 if t.dtype == torch.float8_e4m3fn else t.dtype).zero_()
        self._copy_masters(self.state)

    def _given_state(self, state):
        layout = self._layout()
        if set(state) != set(layout):
            raise ValueError(f'state must hold {sorted(layout)}, got {sorted(state)}')
        for name, (n, dtype) in layout.items():
            t = state[name]
            if t.dtype != dtype or tuple(t.shape) != (n,) or not t.is_contiguous() or t.device != self.device:
                raise ValueError(f'{name} must be a contiguous {dtype} [{n}] on {self.device}')
            if t.data_ptr() % 16:
                raise ValueError(f'{name} must begin at a multiple of 16 bytes')
        return dict(state)

    def part(self, buffer, i):
        """Parameter i's values of a state buffer (not of scales), as a view of the parameter's shape and strides."""
        p = self.params[i]
        return buffer[self.offsets[i]:self.offsets[i] + self._numels[i]].as_strided(
            p.shape, p.stride(), buffer.storage_offset() + self.offsets[i])

    def scales(self, buffer, i):
        """Parameter i's scales of a buffer of them."""
        seg = _ext.ADAMW_SEG
        return buffer[self.offsets[i] // seg:(self.offsets[i] + self._numels[i] + seg - 1) // seg]

    def set_grads(self, grads):
        """Use these gradients from the next step on."""
        self._table.set_grads(list(grads))

    def step(self, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, grad_scale=None):
        """One step, the ``step``-th (from 1).  ``grad_scale``: a float32 GPU scalar that gradients are multiplied
        by.  For a captured graph ``step`` may be an int64 GPU scalar and ``lr`` a float32 one, whose values
        are read when the graph runs."""
        _check_rates(lr, betas, eps, weight_decay)
        if isinstance(step, torch.Tensor):
            at, lr = (lr, 0.0) if isinstance(lr, torch.Tensor) else (None, lr)
            self._table.step_later(step, at, lr, betas[0], betas[1], eps, weight_decay, grad_scale)
        elif isinstance(lr, torch.Tensor):
            raise TypeError('lr may be a GPU scalar only where step is one')
        else:
            self._table.step(step, lr, betas[0], betas[1], eps, weight_decay, grad_scale)


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay on the HIP kernel: GPU parameters in fp32, fp16 or bf16, gradients of
    their dtype.  A group's steps are counted together: a parameter that has no gradient in a step is
    left as it is, and the next bias correction counts that step.

    ``state_bits``, ``master_weights`` (for the 16-bit parameters) and ``seed`` as in ``AdamWPlan``.  ``capturable``: the
    count of steps is a GPU scalar, so that ``step`` can be captured into a graph (after one step outside,
    with gradients that keep their memory); ``lr`` may be a float32 GPU scalar then.

    The state dict holds each parameter's part of the flat buffers; 8-bit states load into parameters of the
    same strides alone, as their scales follow the order in memory."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32,
                 master_weights=False, seed=0, capturable=False):
        _check_rates(lr, betas, eps, weight_decay)
        if state_bits not in _NAMES:
            raise ValueError(f'state_bits must be 32 or 8, got {state_bits}')
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError('lr may be a GPU scalar only with capturable=True')
        self._plans = {}      # group -> [(plan, its parameters, picks them from the group's)]
        self._retired, self._retired_scalars = [], []   # plans, and counts and rates, that a captured graph may still use
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights, seed=seed, capturable=capturable, step=0))

    def _seed(self, gi, dtype):
        return self.param_groups[gi]['seed'] + 2 * gi + (dtype == torch.float32)

    def _group_plans(self, gi):
        """``_plans`` of group gi, one a dtype, made of all its parameters."""
        if gi in self._plans:
            return self._plans[gi]
        group = self.param_groups[gi]
        by_dtype = {}
        for i, p in enumerate(group['params']):
            by_dtype.setdefault(p.dtype, []).append(i)
        out = []
        for dtype, at in by_dtype.items():
            together = at[-1] - at[0] + 1 == len(at)
            pick = operator.itemgetter(slice(at[0], at[-1] + 1)) if together else operator.itemgetter(*at)
            params = list(pick(group['params']))
            master = group['master_weights'] and dtype != torch.float32
            plan = AdamWPlan(params, [None] * len(params), state_bits=group['state_bits'], master_weights=master,
                             seed=self._seed(gi, dtype))
            for i, p in enumerate(params):
                mine = {name: (plan.scales if name.endswith('_scale') else plan.part)(buf, i)
                        for name, buf in plan.state.items()}
                for name, t in self.state[p].items():  # of a copied or unpickled optimizer
                    mine[name].copy_(t)
                self.state[p] = mine
            out.append((plan, params, pick))
        self._plans[gi] = out
        return out

    @torch.no_grad()
    def step(self, closure=None, grad_scale=None):
        """One step; ``grad_scale``: a float32 GPU scalar that gradients are multiplied by (a clipping or loss
        scale's factor).  A step by gradients that are not finite is not skipped: their parameters are lost, and
        with 8-bit states the rest of their segments of 256 a step later.  A loop whose loss scale may be too large
        looks at the gradients first, as torch.amp.GradScaler does."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            if not any(p.grad is not None for p in group['params']):
                continue
            plans = self._group_plans(gi)
            if sum(len(params) for _, params, _ in plans) != len(group['params']):
                raise RuntimeError('a group has gained or lost parameters since the first step: make a new optimizer')
            for plan, _, pick in plans:
                plan._table.follow(pick(group['params']))
            if group['capturable']:
                if not isinstance(group['step'], torch.Tensor):
                    group['step'] = torch.tensor(group['step'], dtype=torch.int64, device=plans[0][0].device)
                group['step'].add_(1)
            else:
                group['step'] += 1
            for plan, *_ in plans:
                plan.step(group['step'], lr=group['lr'], betas=group['betas'], eps=group['eps'],
                          weight_decay=group['weight_decay'], grad_scale=grad_scale)
        return loss

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plans = {}
        self.__dict__.setdefault('_retired', [])
        self.__dict__.setdefault('_retired_scalars', [])

    @staticmethod
    def _fit(group, plans):
        """Whether plans that were made for a group are what its options ask for now."""
        followed = [p for _, params, _ in plans for p in params]
        picked = [p for *_, pick in plans for p in pick(group['params'])] if len(followed) == len(group['params']) else []
        return len(picked) == len(followed) and all(map(operator.is_, picked, followed)) and all(
            plan.state_bits == group['state_bits'] and
            plan.master_weights == bool(group['master_weights'] and params[0].dtype != torch.float32)
            for plan, params, _ in plans)

    def load_state_dict(self, state_dict):
        """As torch's.  Values are loaded into the buffers, the count of steps and the GPU scalar ``lr`` that this
        optimizer has, so that a step captured into a graph goes on from them (with the betas, eps, decay and, where
        it is a number, the rate that it was captured with).  Where the loaded options ask for other states
        (``state_bits``, ``master_weights``) or no GPU scalars (``capturable``) these are made anew, and a step has to
        be captured again.  A state dict
        that does not fit is refused, and leaves the optimizer as it is."""
        groups, states, plans = self.param_groups, self.state, self._plans
        super().load_state_dict({'state': {}, 'param_groups': state_dict['param_groups']})
        try:
            loads = self._matched_states(state_dict, states, plans)
        except Exception:  # refused: nothing has been written
            self.param_groups, self.state, self._plans = groups, states, plans
            raise
        rates = {}  # what groups that share a rate's tensor load into it
        for group, was in zip(self.param_groups, groups):
            rates.setdefault(id(was['lr']), set()).add(float(group['lr']))
        for gi, (group, was) in enumerate(zip(self.param_groups, groups)):
            count, lr = was['step'], was['lr']
            if isinstance(count, torch.Tensor) and group['capturable']:
                group['step'] = count.copy_(torch.as_tensor(group['step']))
            elif isinstance(group['step'], torch.Tensor):  # of the saved optimizer, or on another device
                group['step'] = group['step'].to(device=group['params'][0].device, dtype=torch.int64, copy=True)
            if isinstance(lr, torch.Tensor) and group['capturable'] and len(rates[id(lr)]) == 1:
                group['lr'] = lr.copy_(torch.as_tensor(group['lr']))
            elif isinstance(group['lr'], torch.Tensor) and group['params']:
                group['lr'] = group['lr'].to(group['params'][0].device)
            captured = [plan for plan, *_ in plans.get(gi, ()) if plan._table.captured]
            if captured and self._plans.get(gi) is not plans[gi]:
                self._retired += captured
            if captured:
                self._retired_scalars += [old for old, new in ((count, group['step']), (lr, group['lr']))
                                          if isinstance(old, torch.Tensor) and old is not new]
            for plan, params, _ in self._plans.get(gi, ()):
                plan._reseed(self._seed(gi, params[0].dtype))
        for load in loads:
            load()
        for made in self._plans.values():
            for plan, *_ in made:
                plan._table.masters_match()

    def _matched_states(self, state_dict, states, plans):
        """The calls that load what a state dict holds, with plans and states for them: those that there were, where
        they are what the loaded options ask for."""
        saved, loads = state_dict['state'], []
        for gi, (group, old) in enumerate(zip(self.param_groups, state_dict['param_groups'])):
            if not _OPTIONS <= set(old):
                raise ValueError(f'the state dict\'s options lack {sorted(_OPTIONS - set(old))}: of another optimizer?')
            kept = gi in plans and self._fit(group, plans[gi])
            if kept:
                self._plans[gi] = plans[gi]
                self.state.update((p, states[p]) for p in group['params'])
            if not any(k in saved for k in old['params']):
                loads += [plan._start_over for plan, *_ in plans[gi]] if kept else []
                continue
            self._group_plans(gi)
            for p, k in zip(group['params'], old['params']):
                if k not in saved:
                    raise ValueError('the state dict holds some of a group\'s states only')
                mine, theirs = self.state[p], saved[k]
                if set(mine) != set(theirs):
                    raise ValueError(f'the state dict holds {sorted(theirs)}, this optimizer {sorted(mine)}')
                for name, t in mine.items():
                    o = theirs[name]
                    if o.shape != t.shape or o.dtype != t.dtype:
                        raise ValueError(f'{name}: {tuple(o.shape)} {o.dtype} in the state dict, {tuple(t.shape)} {t.dtype} here')
                    if group['state_bits'] == 8 and not _same_layout(o, t):
                        raise ValueError('8-bit states load into parameters of the same strides alone')
                    loads.append(functools.partial(t.copy_, o))
        return loads
