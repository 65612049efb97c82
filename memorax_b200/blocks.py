"""Minimal mirrors of the reference's composition blocks, only as far as the
training-step benchmark needs them: ``GatedResidual`` (x + sigmoid(Dense(x)) *
module(x), blocks/residual.py:33-63), ``PreNorm`` (LayerNorm before the module,
blocks/normalization.py:10-35), ``FFN`` (Dense-gelu-Dense, blocks/ffn.py:11-50)
and ``Stack`` (blocks/stack.py:33-60), with the reference's
``(inputs, done, initial_carry) -> (carry, outputs)`` block signature, plus the
flat-buffer trainer that runs forward, backward, the gradient all-reduce and
the fused Adam kernel; and the parts of a policy over discrete symbols
(``Embedding``, ``CategoricalHead``, ``TokenPolicyNet``) with the optimiser for
a model's own tensors (``AdamW``)."""
from __future__ import annotations

import torch
from torch import nn

from . import _C, ops
from .memoroid import DeltaNetCell, Memoroid, plain


class PreNorm(nn.Module):
    def __init__(self, module, features):
        super().__init__()
        self.module, self.norm = module, nn.LayerNorm(features)

    def forward(self, inputs, done=None, initial_carry=None):
        normed = ops.layer_norm(inputs, self.norm.weight, self.norm.bias, self.norm.eps)
        return self.module(normed, done, initial_carry)


class Dense(nn.Linear):
    """``nn.Linear`` whose bias gradient is this library's fixed-order column sum (``ops.dense``)."""

    def forward(self, x):
        return ops.dense(x, self.weight, self.bias)


class GatedResidual(nn.Module):
    def __init__(self, module, features):
        super().__init__()
        self.module, self.gate = module, Dense(features, features)

    def forward(self, inputs, done=None, initial_carry=None):
        fork = None
        if plain(self.module, PreNorm):   # the norm, the gate and the sum read the same inputs
            norm = self.module.norm
            fork = ops.norm_fork(inputs, norm.weight, norm.bias, norm.eps)
        if fork is not None:
            normed, inputs, gated = fork
            carry, out = self.module.module(normed, done, initial_carry)
        else:
            gated = inputs
            carry, out = self.module(inputs, done, initial_carry)
        if plain(self.gate, Dense):
            return carry, ops.gated_dense(inputs, gated, self.gate, out)
        return carry, ops.gated_residual(inputs, self.gate(gated), out)


class FFN(nn.Module):
    def __init__(self, features, expansion_factor=4):
        super().__init__()
        self.up, self.down = Dense(features, features * expansion_factor), Dense(features * expansion_factor, features)

    def forward(self, inputs, done=None, initial_carry=None):
        return None, self.down(ops.dense_gelu(inputs, self.up) if plain(self.up, Dense) else ops.gelu(self.up(inputs)))


class Stack(nn.Module):
    def __init__(self, blocks):
        super().__init__()
        self.blocks = nn.ModuleList(blocks)

    def forward(self, inputs, done=None, initial_carry=None):
        carries, x = [], inputs
        initial_carry = initial_carry or (None,) * len(self.blocks)
        for block, carry in zip(self.blocks, initial_carry):
            c, x = block(x, done, carry)
            carries.append(c)
        return tuple(carries), x


class GTrXLStyleValueNet(nn.Module):
    """Dense(obs -> d_model) -> [GatedResidual(PreNorm(mixer)), GatedResidual(PreNorm(FFN))] x layers
    -> Dense(d_model -> 1); the reference's "GTrXL-style" composition
    (README.md:119-124) with the attention block replaced by the delta-rule mixer."""

    def __init__(self, obs_dim=128, d_model=512, num_heads=8, head_dim=64, layers=4):
        super().__init__()
        self.embed = Dense(obs_dim, d_model)
        blocks = []
        for _ in range(layers):
            mixer = Memoroid(DeltaNetCell(features=d_model, head_dim=head_dim, num_heads=num_heads))
            blocks += [GatedResidual(PreNorm(mixer, d_model), d_model), GatedResidual(PreNorm(FFN(d_model), d_model), d_model)]
        self.torso = Stack(blocks)
        self.head = nn.Linear(d_model, 1)

    def forward(self, obs, done):
        _, x = self.torso(self.embed(obs), done)
        return self.head(x).squeeze(-1)


class Embedding(nn.Module):
    """Features of a token (networks/embedding.py): its row of ``weight`` times ``scale``; tokens outside of the vocabulary
    (padding) give zeros."""

    def __init__(self, vocab, features, scale=1.0):
        super().__init__()
        self.weight, self.scale = nn.Parameter(torch.randn(vocab, features) / features ** 0.5), scale

    def forward(self, tokens):
        return ops.embedding(tokens, self.weight, self.scale)


class CategoricalHead(nn.Module):
    """A categorical policy (networks/heads.py): logits, and what an update or an acting step needs of them."""

    def __init__(self, features, actions):
        super().__init__()
        self.logits = Dense(features, actions)

    def forward(self, x, actions=None, mask=None, temperature=1.0, top=0):
        """-> ``ops.TokenLogProbs`` of ``actions`` (...) under the policy at ``x`` (..., F)."""
        return ops.token_log_probs(self.logits(x), actions, mask, temperature, top)


class TokenPolicyNet(nn.Module):
    """A policy over discrete observations and actions: embedding -> [GatedResidual(PreNorm(delta rule with positions)),
    GatedResidual(PreNorm(FFN))] x layers -> categorical head; the value network's composition with symbols at both ends."""

    def __init__(self, observations, actions, d_model=512, num_heads=8, head_dim=64, layers=4, rotary_base=10000.0):
        super().__init__()
        self.embed = Embedding(observations, d_model, scale=d_model ** 0.5)
        blocks = []
        for _ in range(layers):
            mixer = Memoroid(DeltaNetCell(features=d_model, head_dim=head_dim, num_heads=num_heads, rotary_base=rotary_base))
            blocks += [GatedResidual(PreNorm(mixer, d_model), d_model), GatedResidual(PreNorm(FFN(d_model), d_model), d_model)]
        self.torso = Stack(blocks)
        self.head = CategoricalHead(d_model, actions)

    def forward(self, observations, done=None, initial_carry=None, **head):
        """``observations`` (B,T) tokens -> (next_carry, ``ops.TokenLogProbs``); ``head``: the head's arguments."""
        carry, x = self.torso(self.embed(observations), done, initial_carry)
        return carry, self.head(x, **head)


class TokenPolicyTrainer:
    """Policy-gradient updates of a :class:`TokenPolicyNet`: the loss is ``-mean(advantage * log_prob) - entropy_coef *
    mean(entropy)``, the optimiser :class:`AdamW` over the network's own parameters (``adamw``: its arguments)."""

    def __init__(self, model, entropy_coef=0.01, check_every=16, **adamw):
        self.model, self.entropy_coef, self.check_every = model, entropy_coef, check_every
        self.optimiser = AdamW(model.parameters(), **adamw)
        self.calls = 0

    def step(self, observations, actions, done, advantage, mask=None):
        self.optimiser.zero_grad()
        _, policy = self.model(observations, done, actions=actions, mask=mask)
        loss = -(advantage * policy.log_prob).mean() - self.entropy_coef * policy.entropy.mean()
        loss.backward()
        self.optimiser.step()
        self.calls += 1                            # (a capturable optimiser's own number is on the device)
        if self.calls % self.check_every == 0 and not torch.cuda.is_current_stream_capturing():
            ops.check_status(observations.device)
        return loss.detach()


class FlatAdamTrainer:
    """Keeps every parameter (bf16) and gradient as a view into one flat buffer so
    that Adam is one kernel launch and the gradient all-reduce works on contiguous
    ranges.  The update itself is applied to an fp32 master copy (optax.adam on the
    reference's fp32 params); the bf16 buffer the model computes with is its rounding,
    rewritten by the same kernel -- a step of lr = 3e-4 is far below a bf16 ulp at |p| = 1.

    The flat gradient is cut into one bucket per top-level block (embedding, each torso block,
    head).  Parameters enter the backward pass without a ``.grad``, so autograd hands over each
    gradient tensor as it is (no add kernel per parameter, no zeroing of the flat buffer); a
    gradient hook copies a bucket's gradients into the flat buffer with one multi-tensor copy the
    moment the last of them has arrived and, with more than one rank, launches that bucket's
    all-reduce, which runs on NCCL's stream underneath the rest of the backward pass; the step
    waits for all buckets before the Adam kernel."""

    def __init__(self, model, lr=3e-4, betas=(0.9, 0.999), eps=1e-8, process_group=None, world_size=1,
                 overlap_allreduce=True):
        self.model, self.lr, self.betas, self.eps = model, lr, betas, eps
        self.group, self.world = process_group, world_size
        params = [p for p in model.parameters()]
        total = sum(p.numel() for p in params)
        padded = (total + 7) // 8 * 8
        dev = params[0].device
        self.flat = torch.zeros(padded, dtype=torch.bfloat16, device=dev)
        self.flat_grad = torch.zeros(padded, dtype=torch.bfloat16, device=dev)
        off = 0
        offsets = {}
        for p in params:
            n = p.numel()
            self.flat[off:off + n].copy_(p.data.reshape(-1))
            p.data = self.flat[off:off + n].view_as(p)
            offsets[p] = (off, off + n)
            off += n
        self.master = self.flat.float()
        self.m = torch.zeros(padded, dtype=torch.float32, device=dev)
        self.v = torch.zeros(padded, dtype=torch.float32, device=dev)
        self.step_count = 0
        self.check_every = 16
        self.num_params = total
        # ---- gradient buckets: contiguous ranges of the flat buffer, one per top-level block
        self.buckets = []          # (lo, hi, number of parameters)
        self._bucket_params = []   # per bucket: (parameters, their views into the flat gradient)
        self._pending, self._handles = [], []
        self._params = params
        self._reduce_in_hooks = world_size > 1 and overlap_allreduce
        for child in self._top_level_blocks(model):
            ps = [p for p in child.parameters()]
            if not ps:
                continue
            lo, hi = min(offsets[p][0] for p in ps), max(offsets[p][1] for p in ps)
            index = len(self.buckets)
            self.buckets.append((lo, hi, len(ps)))
            self._bucket_params.append((ps, [self.flat_grad[offsets[p][0]:offsets[p][1]].view_as(p) for p in ps]))
            for p in ps:
                p.register_post_accumulate_grad_hook(self._make_hook(index))
        covered = sorted((lo, hi) for lo, hi, _ in self.buckets)
        assert covered[0][0] == 0 and covered[-1][1] == total and all(
            a[1] == b[0] for a, b in zip(covered, covered[1:])), "buckets must tile the flat gradient"

    @staticmethod
    def _top_level_blocks(model):
        for child in model.children():
            if isinstance(child, Stack):
                yield from child.blocks
            else:
                yield child

    def _make_hook(self, index):
        def hook(_param):
            self._pending[index] -= 1
            if self._pending[index] == 0:
                ps, views = self._bucket_params[index]
                torch._foreach_copy_(views, [p.grad for p in ps])
                for p in ps:
                    p.grad = None
                if self._reduce_in_hooks:
                    import torch.distributed as dist
                    lo, hi, _ = self.buckets[index]
                    self._handles.append(dist.all_reduce(self.flat_grad[lo:hi], group=self.group, async_op=True))
        return hook

    def step(self, obs, done, target):
        for p in self._params:
            p.grad = None
        self._pending = [n for _, _, n in self.buckets]
        self._handles = []
        value = self.model(obs, done)
        loss = 0.5 * (value.float() - target).square().mean()     # VNetwork.loss, heads.py:114-117
        loss.backward()
        assert not any(self._pending), "a gradient bucket never filled (a parameter received no gradient)"
        if self.world > 1:
            if self._reduce_in_hooks:
                for handle in self._handles:
                    handle.wait()
                assert len(self._handles) == len(self.buckets), "a gradient bucket was never reduced"
            else:
                import torch.distributed as dist
                dist.all_reduce(self.flat_grad, group=self.group)
        self.step_count += 1
        ops.adam_step(self.flat, self.flat_grad, self.m, self.v, self.step_count, self.lr, self.betas, self.eps,
                      grad_scale=1.0 / self.world, master=self.master)
        if self.step_count % self.check_every == 0:
            ops.check_status(self.flat.device)   # a bounded wait that gave up inside the mixer kernels
        return loss.detach()


class AdamW:
    """AdamW (``optax.adamw``) over a model's own tensors, one launch a step for as many as 700 of a type; with ``t`` the number of
    steps taken:
    ``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g^2``,
    ``p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)``, in float32.

    ``params``: contiguous float32, bfloat16 or float16 tensors of one device, each memory once.  ``master``: ``True`` (float32
    copies are made of the 16-bit parameters) or a list of float32 tensors that take the update; the parameters then hold their
    rounding.  Float32 parameters, of which a list may hold some, take the update themselves: their place in ``master`` is ``None``.  ``state_bits=8``: the moments are 8-bit floats (e4m3) with a float32 scale for every 256 elements, of the second
    its root; a gradient that is not finite then spoils the 256 moments it is among.  ``capturable=True``: number of steps and
    ``lr`` live on the device (``lr`` is a tensor that may be written between steps), for steps in a captured graph; without it
    a step refuses to be captured.

    The moments are one buffer each, a tensor's from ``starts[i]`` on: ``m`` and ``v`` are the float32 buffers, or pairs of
    8-bit codes and scales.  :meth:`moments` gives their values tensor by tensor."""

    def __init__(self, params, lr=3e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, master=None, capturable=False):
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1) or eps < 0:
            raise ValueError(f"betas must be in [0, 1) and eps not negative, got {betas} and {eps}")
        self._given = list(params)
        if master is True:
            master = [None if p.dtype == torch.float32 else p.float() for p in self.params]
        self.master = master if master is None else list(master)
        self.betas, self.eps, self.weight_decay, self.state_bits, self.capturable = tuple(betas), eps, weight_decay, state_bits, capturable
        self._native = _C.AdamW(self._given, self.master, state_bits)
        self.starts = self._native.starts
        self._step, self.lr = 0, lr
        self._count = self._now = None
        if capturable:
            device = self._given[0].device
            self.lr = lr if isinstance(lr, torch.Tensor) else torch.tensor(float(lr), device=device)
            if self.lr.dtype != torch.float32 or self.lr.device != device or self.lr.numel() != 1:
                raise ValueError("lr must be one float32 on the parameters' device")
            self._count = torch.zeros((), dtype=torch.int64, device=device)
            self._now = torch.zeros(3, device=device)

    def _moment(self, which):
        held, scale = getattr(self._native, which), getattr(self._native, which + "_scale")
        return held if scale is None else (held, scale)

    #: the parameters, without the graph
    params = property(lambda self: [p.detach() for p in self._given])
    m = property(lambda self: self._moment("m"))
    v = property(lambda self: self._moment("v"))

    @property
    def step_count(self):
        return int(self._count) if self.capturable else self._step

    def step(self, grads=None, grad_scale=1.0):
        """One update from ``grads`` (of the parameters' type or float32; ``None`` leaves a parameter as it is), or from each
        parameter's ``.grad``, times ``grad_scale``."""
        if self.capturable:
            self._native.step(grads, 0.0, *self.betas, self.eps, self.weight_decay, grad_scale, 0, self._count, self.lr, self._now)
            return
        self._native.step(grads, self.lr, *self.betas, self.eps, self.weight_decay, grad_scale, self._step + 1, None, None, None)
        self._step += 1

    def zero_grad(self):
        for p in self._given:
            p.grad = None

    def moments(self):
        """``(m, v)``: lists of float32 tensors of the parameters' shapes (copies where the moments are held in 8 bits)."""
        if self.state_bits == 32:
            return self._native.cut(self.m), self._native.cut(self.v)
        values = lambda held: (held[0].float().view(-1, 256) * held[1][:, None]).flatten()
        return self._native.cut(values(self.m)), self._native.cut(values(self.v).square())

    def load(self, m, v, step, master=None):
        """Takes over moments (as :meth:`moments` gives them) and the number of steps behind them.  ``master``: ``None`` leaves the
        float32 copies as they are, ``True`` makes them again from the parameters (after these were loaded), a list of tensors is
        taken over."""
        flats = []
        for given in (m, v):
            flat, given = torch.zeros(self._native.m.numel(), device=self._given[0].device), list(given)
            if len(given) != len(self._given) or any(x.shape != p.shape for x, p in zip(given, self._given)):
                raise ValueError("moments must be of the parameters' shapes")
            torch._foreach_copy_(self._native.cut(flat), given)
            flats.append(flat)
        copies = self._copies(master)
        for mine, flat, root in zip((self.m, self.v), flats, (False, True)):
            if self.state_bits == 32:
                mine.copy_(flat)
            else:
                for to, x in zip(mine, _hold(flat.sqrt() if root else flat, root)):
                    to.copy_(x)
        self._take(copies, step)

    def state_dict(self):
        """What is held, as it is held: the moments, the float32 copies (``None`` without), the number of steps."""
        copy = lambda held: tuple(x.clone() for x in held) if isinstance(held, tuple) else held.clone()
        return {"m": copy(self.m), "v": copy(self.v), "master": None if self.master is None else [None if x is None else x.clone() for x in self.master],
                "step": self.step_count, "state_bits": self.state_bits}

    def load_state_dict(self, state):
        """Takes over what :meth:`state_dict` gave; nothing is written where a part of it does not fit.  Where the state has no float32
        copies they are made again from the parameters, which are loaded before."""
        if state["state_bits"] != self.state_bits:
            raise ValueError(f"the state has {state['state_bits']} bits, this optimiser {self.state_bits}: use moments() and load()")
        pairs = []
        for mine, given in ((self.m, state["m"]), (self.v, state["v"])):
            pairs += zip(mine if isinstance(mine, tuple) else (mine,), given if isinstance(given, tuple) else (given,), strict=True)
        for to, x in pairs:
            if to.shape != x.shape or to.dtype != x.dtype:
                raise ValueError(f"a moment of {tuple(x.shape)} {x.dtype} for one of {tuple(to.shape)} {to.dtype}")
        master = state.get("master")
        copies = self._copies(master if master is not None or self.master is None else True)
        for to, x in pairs:
            to.copy_(x)
        self._take(copies, state["step"])

    def _copies(self, master):
        """Pairs (float32 copy, what it is to hold); ``master`` as :meth:`load` takes it."""
        if master is None:
            return []
        if self.master is None:
            raise ValueError("float32 copies for an optimiser that was built without (master)")
        given = self.params if master is True else list(master)
        if master is True:
            given = [None if to is None else x for to, x in zip(self.master, given)]
        if len(given) != len(self.master) or any((x is None) != (to is None) or (to is not None and x.numel() != to.numel()) for to, x in zip(self.master, given)):
            raise ValueError("float32 copies must be of the 16-bit parameters and their sizes")
        return [(to, x.reshape(to.shape)) for to, x in zip(self.master, given) if to is not None]

    def _take(self, copies, step):
        with torch.no_grad():
            for to, x in copies:
                to.copy_(x)
        self._step = int(step)
        if self.capturable:
            self._count.fill_(self._step)


def _hold(x, root):
    """A buffer of whole 256s as 8-bit floats and scales, the way the kernel holds it (adamw.cu)."""
    rows = x.view(-1, 256)
    top = rows.abs().amax(-1, keepdim=True)
    top = torch.where(top < 2.0 ** -100, 0.0, top)
    held = rows * torch.where(top > 0, 448.0 / top, 0.0)
    if root:
        held = torch.where((top > 0) & (rows > 0), held.clamp_min(2.0 ** -9), held)
    return held.to(torch.float8_e4m3fn).flatten(), (top / 448.0).flatten()
