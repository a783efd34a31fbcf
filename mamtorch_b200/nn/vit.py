"""Putting MAM layers into a transformer MLP block, the way the reference's ViT example does it.

The reference fine-tunes a Hugging Face ViT-B/16 after replacing the two dense layers of every MLP
block (`vit.encoder.layer.{i}.intermediate.dense`, `.output.dense`) by `mamtorch.nn.FullyConnected`
that start from the dense weights (`examples/vitb16_imagenet1k/utils.py:23-77`), and steps the
vanishing-contribution schedule of every MAM layer once per optimiser step
(`examples/vitb16_imagenet1k/vit_training.py:521-524`).  This module carries that call pattern,
without the example's dependence on a checkpoint or a dataset:

  * `swap_linear_for_mam` / `mlp_dense_paths`  the layer replacement (works on any module tree);
  * `vcon_step_all`                            one schedule step for every MAM layer of a model;
  * `MAMMlpBlock`                              LayerNorm -> MAM(d, 4d) -> GELU -> MAM(4d, d) + residual,
                                               the MLP half of a ViT encoder layer, for runs on
                                               synthetic tokens; with `fused=True` what stands between
                                               the MAM layers, dropout included, runs in this library's
                                               own kernels;
  * `MAMMlpStack`                              such blocks one after the other with the encoder's final
                                               norm: each residual addition, its dropout and the norm of
                                               the next block in one pass;
  * `GraphedStep`                              forward + backward of a module captured in one CUDA
                                               graph on static buffers (the kernels take the current
                                               stream and allocate through torch's caching allocator,
                                               so they capture like any other torch operator).
"""
from __future__ import annotations

import torch
from torch import nn

from . import functional as MF
from .v4.fullyconnected import FullyConnected

__all__ = ["mlp_dense_paths", "swap_linear_for_mam", "vcon_step_all", "mam_layers", "MAMMlpBlock", "MAMMlpStack",
           "GraphedStep"]


def mlp_dense_paths(num_layers: int = 12, intermediate: bool = True, output: bool = True,
                    prefix: str = "vit.encoder.layer") -> list[str]:
    """Attribute paths of the MLP dense layers of a Hugging Face ViT, as `generate_paths` builds
    them in the reference (`examples/vitb16_imagenet1k/utils.py:23-48`).  A negative `num_layers`
    selects the last |num_layers| of 12 encoder layers, as there."""
    layers = range(num_layers) if num_layers >= 0 else range(12 + num_layers, 12)
    paths = []
    if intermediate:
        paths += [f"{prefix}.{i}.intermediate.dense" for i in layers]
    if output:
        paths += [f"{prefix}.{i}.output.dense" for i in layers]
    return paths


def _resolve(model: nn.Module, path: str):
    parent = model
    parts = path.split(".")
    for p in parts[:-1]:
        parent = getattr(parent, p)
    return parent, parts[-1]


def swap_linear_for_mam(model: nn.Module, paths, vcon_steps: int = 0, vcon_type: str = "linear", splits: int = 1,
                        train_mam_only: bool = False, **mam_kwargs) -> nn.Module:
    """Replaces the `nn.Linear` at every path by a `FullyConnected` that takes over its weight and
    bias (`add_mam_to_ViT`, `examples/vitb16_imagenet1k/utils.py:67-77`).  With `vcon_steps > 0` the
    new layers start as the dense layers they replace (beta = 1) and turn into MAM layers over that
    many `vcon_step()` calls."""
    for path in paths:
        parent, attr = _resolve(model, path)
        lin = getattr(parent, attr)
        if not isinstance(lin, nn.Linear):
            raise TypeError(f"{path} is a {type(lin).__name__}, not an nn.Linear")
        mam = FullyConnected(lin.in_features, lin.out_features, bias=lin.bias is not None, vcon_steps=vcon_steps,
                             vcon_type=vcon_type, splits=splits, train_mam_only=train_mam_only,
                             device=lin.weight.device, dtype=lin.weight.dtype, **mam_kwargs)
        mam.weight.data = lin.weight.data
        if lin.bias is not None:
            mam.bias.data = lin.bias.data
        setattr(parent, attr, mam)
    return model


def mam_layers(model: nn.Module):
    """Every MAM fully-connected layer of a model, in module order."""
    return [m for m in model.modules() if isinstance(m, FullyConnected)]


def vcon_step_all(model: nn.Module) -> None:
    """One step of the vanishing-contribution schedule on every MAM layer: what the reference's
    training loop does after each optimiser step (`vit_training.py:521-524`)."""
    for layer in mam_layers(model):
        layer.vcon_step()


class _DropSeeds(nn.Module):
    """Seeds for the dropout of a module.  Eagerly they are numbers from torch's CPU generator.  Inside a graph capture a
    number would repeat one mask at every replay, so there a device counter is advanced, which the graph does again each
    time it runs, and a number drawn at the capture is added: deep copies of a module copy its counter."""

    def __init__(self, device=None):
        super().__init__()
        self.register_buffer("counter", torch.tensor([MF.fresh_drop_seed()], dtype=torch.int64, device=device),
                             persistent=False)

    def forward(self):
        if not (self.counter.is_cuda and torch.cuda.is_current_stream_capturing()):
            return MF.fresh_drop_seed()
        self.counter.add_(0x632BE59BD9B4E019)
        return self.counter + MF.fresh_drop_seed()


class MAMMlpBlock(nn.Module):
    """The MLP half of a pre-norm transformer encoder layer with MAM dense layers:
    x + MAM_2(GELU(MAM_1(LayerNorm(x)))), shapes [..., hidden] -> [..., hidden].

    ViT-B/16: hidden 768, intermediate 3072, 197 tokens per image.

    `fused=True` runs norm, GELU and residual in this library's kernels (equal to torch's up to rounding) and allows
    `drop_rate`: dropout behind the GELU and before the residual, in training, with masks that are never stored.  `norm` then
    lends its weight, bias and eps; it and `act` are not called as modules (their hooks do not run)."""

    def __init__(self, hidden: int = 768, intermediate: int = 3072, vcon_steps: int = 0, vcon_type: str = "linear",
                 store_args: bool = False, residual: bool = True, layer_norm_eps: float = 1e-12, device=None,
                 dtype=None, fused: bool = False, drop_rate: float = 0.0):
        super().__init__()
        if not 0.0 <= drop_rate < 1.0:
            raise ValueError(f"drop_rate must be in [0, 1), not {drop_rate}")
        if drop_rate > 0 and not fused:
            raise ValueError("drop_rate needs fused=True")
        self.norm = nn.LayerNorm(hidden, eps=layer_norm_eps, device=device, dtype=dtype)
        self.fc1 = FullyConnected(hidden, intermediate, vcon_steps=vcon_steps, vcon_type=vcon_type,
                                  store_args=store_args, device=device, dtype=dtype)
        self.act = nn.GELU()
        self.fc2 = FullyConnected(intermediate, hidden, vcon_steps=vcon_steps, vcon_type=vcon_type,
                                  store_args=store_args, device=device, dtype=dtype)
        self.residual = residual
        self.fused = fused
        self.drop_rate = drop_rate
        self.drop_seeds = _DropSeeds(device) if drop_rate > 0 else None

    def drop_args(self):
        """(rate, seed) of the next dropout: nothing outside training."""
        if self.drop_seeds is None or not self.training:
            return 0.0, None
        return self.drop_rate, self.drop_seeds()

    def mlp(self, h: torch.Tensor) -> torch.Tensor:
        """The MAM layers on a normalised input, with the fused activation between them."""
        return self.fc2(MF.gelu(self.fc1(h), *self.drop_args()))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.fused:
            y = self.mlp(MF.layer_norm(x, self.norm.weight, self.norm.bias, self.norm.eps))
            rate, seed = self.drop_args()
            if not self.residual and rate == 0.0:
                return y
            return MF.dropout(y, rate, seed, residual=x if self.residual else None)
        y = self.fc2(self.act(self.fc1(self.norm(x))))
        return x + y if self.residual else y

    def vcon_step(self) -> None:
        self.fc1.vcon_step()
        self.fc2.vcon_step()


class MAMMlpStack(nn.Module):
    """`depth` fused MLP blocks and the final norm of the encoder (`vit.layernorm` of a Hugging Face ViT):
    LayerNorm(block_depth(... block_1(x))).  The residual stream and the next norm's output come out of one pass, so the
    blocks and norms are not called as modules themselves (the MAM layers in them are)."""

    def __init__(self, depth: int, hidden: int = 768, intermediate: int = 3072, layer_norm_eps: float = 1e-12,
                 drop_rate: float = 0.0, device=None, dtype=None, **block_kwargs):
        super().__init__()
        if depth < 1:
            raise ValueError("depth must be at least 1")
        self.blocks = nn.ModuleList(
            MAMMlpBlock(hidden, intermediate, layer_norm_eps=layer_norm_eps, device=device, dtype=dtype, fused=True,
                        drop_rate=drop_rate, **block_kwargs) for _ in range(depth))
        if not self.blocks[0].residual:
            raise ValueError("the blocks of a stack have residuals")
        self.norm = nn.LayerNorm(hidden, eps=layer_norm_eps, device=device, dtype=dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        norms = [block.norm for block in self.blocks] + [self.norm]
        h = MF.layer_norm(x, norms[0].weight, norms[0].bias, norms[0].eps)
        for block, norm in zip(self.blocks, norms[1:]):
            h, x = MF.dropout_add_layer_norm(block.mlp(h), x, norm.weight, norm.bias, norm.eps, *block.drop_args())
        return h

    def vcon_step(self) -> None:
        for block in self.blocks:
            block.vcon_step()


class GraphedStep:
    """Forward + backward of `module` on inputs of one fixed shape, captured once in a CUDA graph.

        step = GraphedStep(block, example_x, example_grad_out)
        y = step(x, grad_out)          # replays: y, step.grad_input and the parameters' .grad are refreshed

    Parameter gradients are written into the same `.grad` tensors on every replay (zeroed inside the
    graph), so an optimiser can read them after the call.  The blend weights alpha / beta of a MAM
    layer are kernel arguments and therefore frozen into the graph: capture after the
    vanishing-contribution schedule has ended, or call `recapture()` after each `vcon_step()`.
    """

    def __init__(self, module: nn.Module, example_input: torch.Tensor, example_grad_output: torch.Tensor,
                 warmup: int = 3):
        if not example_input.is_cuda:
            raise ValueError("GraphedStep needs CUDA tensors")
        self.module = module
        self.x = example_input.detach().clone().requires_grad_()
        self.gy = example_grad_output.detach().clone()
        self.warmup = warmup
        self.graph = None
        self.y = None
        self.grad_input = None
        self.recapture()

    def _run(self):
        for p in self.module.parameters():
            if p.grad is not None:
                p.grad.zero_()
        if self.x.grad is not None:
            self.x.grad.zero_()
        y = self.module(self.x)
        y.backward(self.gy)
        return y

    def recapture(self) -> None:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(self.warmup):   # allocates the .grad tensors and warms the allocator
                self._run()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            y = self._run()
        self.y = y.detach()
        self.grad_input = self.x.grad

    def __call__(self, x: torch.Tensor, grad_output: torch.Tensor) -> torch.Tensor:
        self.x.data.copy_(x)
        self.gy.copy_(grad_output)
        self.graph.replay()
        return self.y
