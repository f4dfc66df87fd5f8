"""Low-rank adapters of many requests beside shared projections, on gfx950.

  LowRankAdapters  the adapters of one projection: adapters(x, base, plan) is base[t] +
                   scale[a] * (x[t] down[a]^T) up[a]^T for each token t of adapter a
  AdapterPlan      which token has which adapter, sorted once for all projections of a batch
  AdaptedLinear    a projection (int8.Int8Linear, mxfp4.Mxfp4Linear, nn.Linear) with them
  adapt_transformer  puts them beside projections of a transformer

  requests = adapt_transformer(transformer, {"transformer_blocks.1.attn.to_qkv": adapters, ..})
  requests.plan = AdapterPlan(indices, len(adapters))    # indices [batch, tokens], -1: none
  transformer(..)                                        # fused blocks too

Products and sums are fp32; the output is rounded once more, on top of base's own
rounding. Inference only: inputs that require a gradient are refused.
"""
from __future__ import annotations

import functools
from array import array

import torch
from torch import nn

from . import _lib
from .attention import _DTYPES
from .cache import _clash
from .int8 import Int8Linear
from .mxfp4 import Mxfp4Linear

MAX_ADAPTERS, MAX_RANK = 1000, 128


class AdapterPlan:
    """The tokens of a batch by adapter. indices: int32 or int64 of any shape, on the GPU, one
    for each token; one outside [0, adapters) stands for no adapter. It is not copied to
    the host. `update` takes other indices of the same number of tokens into the same
    memory, which captured graphs that use the plan read at their replay."""

    def __init__(self, indices, adapters):
        adapters = int(adapters)
        if not 0 < adapters <= MAX_ADAPTERS:
            raise ValueError(f"a plan has 1 to {MAX_ADAPTERS} adapters, got {adapters}")
        self._check(indices)
        self.tokens, self.adapters = indices.numel(), adapters
        if self.tokens >= 1 << 24:
            raise RuntimeError(f"{self.tokens} tokens are not supported by the HIP adapters (below 2^24)")
        _lib.check_device(indices)
        tiles = _lib.load().lr_adapter_tiles(self.tokens, adapters)
        self.order = torch.empty(self.tokens, dtype=torch.int32, device=indices.device)
        self.tiles = torch.empty((tiles, 4), dtype=torch.int32, device=indices.device)
        self.update(indices)

    @staticmethod
    def _check(indices):
        if indices.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"indices must be int32 or int64, got {indices.dtype}")

    def update(self, indices):
        self._check(indices)
        if indices.numel() != self.tokens:
            raise ValueError(f"the plan has {self.tokens} tokens, got {indices.numel()} indices")
        _lib.same_device(self.order, indices=indices)
        if indices.dtype == torch.int64:
            # Clamped before the conversion, which would wrap what lies past 32 bits.
            indices = indices.clamp(-1, self.adapters).to(torch.int32)
        indices = indices.contiguous()
        _lib.launch(self.order, "lr_adapter_plan", indices.data_ptr(), self.tokens, self.adapters, self.order.data_ptr(),
                    self.tiles.data_ptr())
        return self

    def rows(self, keep, batch=1):
        """The plan of the tokens `keep` (numbers on the GPU) of each of `batch` sequences that this one is of."""
        # The adapter of each place of the order, then of each token.
        sorted_by = torch.repeat_interleave(self.tiles[:, 0], self.tiles[:, 2], output_size=self.tokens)
        indices = torch.empty_like(sorted_by).scatter_(0, self.order.long(), sorted_by)
        return AdapterPlan(indices.view(batch, self.tokens // batch)[:, keep], self.adapters)


def _copies(k, step, odd):
    """Whether the kernels copy rows of k columns `step` elements apart first: not whole ones, or 16
    bytes or a multiple apart, or ones that overlap, or of an x that lies at an odd place."""
    return bool(odd or k % 8 or step % 8 or step >= 1 << 30 or 0 < step < k)


@functools.lru_cache(maxsize=4096)
def _workspace(device, tokens, n, k, rank, adapters, step, odd):
    nbytes = array("q", [0])
    with torch.cuda.device(device):
        _lib.call("lr_adapter_workspace", tokens, n, k, rank, adapters, int(_copies(k, step, odd)),
                  nbytes.buffer_info()[0])
    return nbytes[0]


class LowRankAdapters(nn.Module):
    """The adapters of a projection from in_features to out_features: down [adapters, rank,
    in_features], up [adapters, out_features, rank], bf16 or fp16, and scale, a number or
    [adapters]. Adapters of lower rank than the others have zeros in down behind theirs. How a
    call is laid over the GPU follows from the number of adapters held, not of those in use.

    Buffers: `down` and `up` with their rows filled up with zeros to multiples of 8, and
    `scale` float32 [adapters]. Calls after a move to another type (model.to(torch.bfloat16), which
    takes scale along) are refused: make the adapters of the type they are to have, last.
    """

    def __init__(self, down, up, scale=1.0):
        super().__init__()
        if down.dim() != 3 or up.dim() != 3 or down.shape[0] != up.shape[0] or down.shape[1] != up.shape[2]:
            raise ValueError("expected down [adapters, rank, in_features] and up [adapters, out_features, rank], "
                             f"got {tuple(down.shape)} and {tuple(up.shape)}")
        if down.dtype != up.dtype or down.device != up.device:
            raise ValueError("down and up must have one dtype and device")
        if down.dtype not in _DTYPES:
            raise RuntimeError(f"dtype {down.dtype} is not supported by the HIP adapters (bfloat16 or float16)")
        self.adapters, self.rank, self.in_features = down.shape
        self.out_features = up.shape[1]
        if min(down.shape) == 0 or self.out_features == 0:
            raise ValueError("adapters, rank, in_features and out_features must be positive")
        if self.rank > MAX_RANK or self.adapters > MAX_ADAPTERS:
            raise RuntimeError(f"{self.adapters} adapters of rank {self.rank} are not supported by the HIP adapters "
                               f"(at most {MAX_ADAPTERS} of {MAX_RANK})")
        scale = torch.as_tensor(scale, dtype=torch.float32, device=down.device).detach()
        if scale.dim() > 1 or (scale.dim() == 1 and scale.shape[0] != self.adapters):
            raise ValueError("scale must be a number or [adapters]")

        def rows(t):
            return nn.functional.pad(t.detach(), (0, -t.shape[-1] % 8)).contiguous()

        self.register_buffer("down", rows(down))
        self.register_buffer("up", rows(up))
        self.register_buffer("scale", scale.expand(self.adapters).contiguous())

    def __len__(self):
        return self.adapters

    def forward(self, x, base, plan, *, out=None):
        """base [.., out_features] plus the adapters' products with x [.., in_features], a new
        tensor like base, or `out`, contiguous, which may be base."""
        x_shape, base_shape = x.shape, base.shape
        if x_shape[-1] != self.in_features or base_shape[-1] != self.out_features or x_shape[:-1] != base_shape[:-1]:
            raise ValueError(f"expected x [.., {self.in_features}] and base [.., {self.out_features}], "
                             f"got {tuple(x_shape)} and {tuple(base_shape)}")
        buffers = self._buffers
        down, up, scale = buffers["down"], buffers["up"], buffers["scale"]
        if x.dtype != down.dtype or base.dtype != down.dtype or up.dtype != down.dtype or scale.dtype != torch.float32:
            raise ValueError(f"x and base must be of the adapters' dtype, {down.dtype} (scale float32), "
                             f"got {x.dtype} and {base.dtype}")
        if down.dtype not in _DTYPES:
            raise RuntimeError(f"dtype {down.dtype} is not supported by the HIP adapters (bfloat16 or float16)")
        if torch.is_grad_enabled() and (x.requires_grad or base.requires_grad or (out is not None and out.requires_grad)):
            raise RuntimeError("gradients are not supported by the HIP adapters: call them under torch.no_grad()")
        tokens = x.numel() // self.in_features
        if plan.tokens != tokens or plan.adapters != self.adapters:
            raise ValueError(f"the plan has {plan.tokens} tokens of {plan.adapters} adapters, "
                             f"these are {tokens} of {self.adapters}")
        if out is not None:
            if out.shape != base.shape or out.dtype != base.dtype or not out.is_contiguous():
                raise ValueError("out must be contiguous, like base")
            same = out.data_ptr() == base.data_ptr() and base.is_contiguous()
            if _clash((out,), (None if same else base, x)):   # (adapters and plan: by the call)
                raise ValueError("out must be base itself or memory of its own")
        _lib.check_device(x)
        _lib.same_device(x, base=base, down=down, plan=plan.order, out=out)
        rows = x if len(x_shape) == 2 else x.reshape(tokens, self.in_features)
        onto = base if len(base_shape) == 2 else base.reshape(tokens, self.out_features)
        x_step, column = rows.stride()
        if column != 1 and self.in_features > 1:
            rows = rows.contiguous()
            x_step = self.in_features
        elif tokens == 1:
            x_step = self.in_features   # (any stride; it is not used)
        base_step, column = onto.stride()
        if column != 1 and self.out_features > 1:
            onto = onto.contiguous()
            base_step = self.out_features
        if out is None:
            out = base.new_empty(base_shape)
        x_at = rows.data_ptr()
        nbytes = _workspace(x.get_device(), tokens, self.out_features, self.in_features, self.rank, self.adapters, x_step,
                            x_at & 15)
        ws = _lib.workspace(x, nbytes) if nbytes else None   # held until the launch
        _lib.launch(x, "lr_adapter_add", x_at, x_step, down.data_ptr(), up.data_ptr(),
                    scale.data_ptr(), onto.data_ptr(), base_step, out.data_ptr(), self.out_features,
                    _DTYPES[down.dtype], tokens, self.out_features, self.in_features, self.rank, self.adapters,
                    plan.order.data_ptr(), plan.tiles.data_ptr(), _lib.ptr(ws), nbytes)
        return out


class Requests:
    """What the adapted projections of a transformer share: the plan of the batch that goes
    through it, or None for none of their adapters. Blocks that Flash runs on selected rows
    have the plan of those rows meanwhile (flash.configure_flash)."""

    def __init__(self, plan=None):
        self.plan = plan


def requests_of(modules):
    """The Requests of the adapted projections in some modules, each once."""
    if not AdaptedLinear.any_made:
        return []
    found = (m.requests for module in modules for m in module.modules() if isinstance(m, AdaptedLinear))
    return list({id(requests): requests for requests in found}.values())


_global_hooks = nn.modules.module._global_forward_hooks


def _gives_new_memory(layer):
    """Whether what a call of the layer returns is memory that nothing else holds: a layer whose
    forward is known, with no hook or replaced function that could keep the result or put its own
    in its place."""
    if type(layer) not in (Int8Linear, Mxfp4Linear, nn.Linear):
        return False
    if layer._forward_hooks or _global_hooks or "forward" in layer.__dict__:
        return False
    return type(layer) is not Int8Linear or layer._fused_call() is not None


class AdaptedLinear(nn.Module):
    """A projection with adapters beside it: layer(value), plus the products of the adapters
    that requests.plan gives the tokens. Layers that quantize their input do so as without
    adapters, which see the input itself: fused blocks pass it to this layer unquantized.
    The products are added in the memory of the layer's result where nothing else can hold
    it (an Int8Linear, Mxfp4Linear or nn.Linear without forward hooks), else in new memory."""

    any_made = False   # in this process, also by copy or unpickling

    def __new__(cls, *args, **kwargs):
        AdaptedLinear.any_made = True
        return super().__new__(cls)

    def __init__(self, layer, adapters, requests):
        super().__init__()
        if (layer.in_features, layer.out_features) != (adapters.in_features, adapters.out_features):
            raise ValueError(f"the layer maps {layer.in_features} to {layer.out_features} features, its adapters "
                             f"{adapters.in_features} to {adapters.out_features}")
        self.layer, self.adapters, self.requests = layer, adapters, requests
        self.in_features, self.out_features = layer.in_features, layer.out_features

    @property
    def weight(self):
        return self.layer.weight

    @property
    def bias(self):
        return self.layer.bias

    def forward(self, value):
        y = self.layer(value)
        plan = self.requests.plan
        if plan is None:
            return y
        # In place where nothing else holds y: tokens without an adapter then cost nothing.
        return self.adapters(value, y, plan, out=y if _gives_new_memory(self.layer) and y.is_contiguous() else None)


def adapt_transformer(transformer, adapters):
    """Put adapters beside projections of a transformer: {name of a submodule: its
    LowRankAdapters}. Every name is checked before any is changed. Returns the Requests
    whose plan they follow."""
    requests = Requests()
    layers = {name: transformer.get_submodule(name) for name in adapters}
    for name, layer in layers.items():
        if isinstance(layer, AdaptedLinear):
            raise ValueError(f"{name} has adapters already")
    adapted = {name: AdaptedLinear(layer, adapters[name], requests) for name, layer in layers.items()}
    for name, layer in adapted.items():
        parent, _, child = name.rpartition(".")
        setattr(transformer.get_submodule(parent), child, layer)
    return requests
