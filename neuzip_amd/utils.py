"""Walk a module tree and swap dense Linear layers for compressed ones.

Counterpart of ``_convert`` in neuzip/utils.py:57-68: children whose attribute
name contains ``lm_head`` are left alone, ``nn.Linear`` (and HuggingFace
``Conv1D`` when transformers is importable) are replaced, everything else is
descended into.  Embeddings are not converted by ``_convert``;
``_unroll_convert`` (neuzip/utils.py:41-54) replaces every Linear AND every
Embedding of the tree, ``lm_head`` included.
"""
from __future__ import annotations

import logging

import torch

logger = logging.getLogger(__name__)


def _convertible_types():
    kinds = [torch.nn.Linear]
    try:  # transformers is optional on this platform
        from transformers.pytorch_utils import Conv1D

        kinds.append(Conv1D)
    except Exception:  # pragma: no cover
        pass
    return tuple(kinds)


def _delete_module(module: torch.nn.Module) -> None:
    """Release the dense parameters of a module that has been replaced."""
    for pname in [n for n, _ in module.named_parameters()]:
        setattr(module, pname, None)


def _set_module_by_name(parent: torch.nn.Module, name: str, child: torch.nn.Module) -> None:
    """``parent.a.3.b = child`` for the dotted ``name`` "a.3.b" (neuzip/utils.py:19-31)."""
    *path, leaf = name.split(".")
    holder = parent
    for part in path:
        holder = holder[int(part)] if part.isnumeric() else getattr(holder, part)
    setattr(holder, leaf, child)


def _unroll_convert(manager, module: torch.nn.Module) -> torch.nn.Module:
    """In place: every ``nn.Linear`` becomes a compressed Linear and every
    ``nn.Embedding`` a compressed Embedding (neuzip/utils.py:41-54)."""
    from neuzip_amd.nn import Embedding, Linear

    for name, m in list(module.named_modules()):
        if not name:
            continue
        if isinstance(m, torch.nn.Linear):
            logger.debug("Quantizing %s: %s", name, m)
            _set_module_by_name(module, name, Linear(manager, m))
            _delete_module(m)
        elif isinstance(m, torch.nn.Embedding):
            logger.debug("Quantizing %s: %s", name, m)
            _set_module_by_name(module, name, Embedding(manager, m))
            _delete_module(m)
    return module


def _convert(manager, module: torch.nn.Module, prefix: str = "") -> torch.nn.Module:
    from neuzip_amd.nn import Linear

    kinds = _convertible_types()
    pending = [(module, prefix)]
    while pending:
        parent, path = pending.pop()
        for name, child in list(parent.named_children()):
            dotted = f"{path}.{name}" if path else name
            if "lm_head" in name:
                continue
            if isinstance(child, kinds):
                logger.debug("Converting %s: %s", dotted, child)
                setattr(parent, name, Linear(manager, child))
                _delete_module(child)
            else:
                pending.append((child, dotted))
    return module


def _heads(module: torch.nn.Module, *marks: str) -> set:
    """The modules that stand in or below a child whose name contains one of ``marks`` (``lm_head``)."""
    marks = marks or ("lm_head",)
    heads, pending, seen = set(), [module], set()
    while pending:
        parent = pending.pop()
        if parent in seen:
            continue
        seen.add(parent)
        for name, child in parent._modules.items():  # every name: named_children gives a module once
            if child is None:
                continue
            if any(mark in name for mark in marks):
                heads.update(child.modules())
            else:
                pending.append(child)
    return heads


def _replace(module: torch.nn.Module, prefix: str, make, made, kept) -> torch.nn.Module:
    """In place: children (at any depth) for which ``make(child)`` is not None become what it gives, those in ``kept``
    aside.  A module that stands in several places is replaced once."""
    for name, child in list(module._modules.items()):
        dotted = f"{prefix}.{name}" if prefix else name
        if child is None or child in kept:
            continue
        if child not in made:
            new = make(child)
            if new is not None:
                logger.debug("Converting %s: %s", dotted, child)
                made[child] = new
                _delete_module(child)
        if child in made:
            setattr(module, name, made[child])
        else:
            _replace(child, dotted, make, made, kept)
    return module


def mx_convert(module: torch.nn.Module, prefix: str = "") -> torch.nn.Module:
    """In place: the ``nn.Linear`` layers that ``Manager.convert`` would compress
    (those whose attribute name contains ``lm_head`` are left alone, wherever else
    they stand too) are held in microscaled 4 bits instead, with their weights
    frozen.  A layer that stands in several places is converted once."""
    from neuzip_amd.nn import MXLinear

    return _replace(module, prefix, lambda m: MXLinear(m) if isinstance(m, torch.nn.Linear) else None, {},
                    _heads(module))


def fp8_convert(module: torch.nn.Module, prefix: str = "", block_rows: int = 128) -> torch.nn.Module:
    """The same with weights in 8 bits: 128 rows of 128 columns share a scale, or with
    ``block_rows=1`` 128 values of a row."""
    from neuzip_amd.nn import FP8Linear

    return _replace(module, prefix, lambda m: FP8Linear(m, block_rows) if isinstance(m, torch.nn.Linear) else None, {},
                    _heads(module))


def fp8_activations(module: torch.nn.Module, skip=(), prefix: str = "") -> torch.nn.Module:
    """In place: what a training step keeps of activations is kept in 8 bits.  Compressed
    Linear layers (``neuzip_amd.nn.Linear``) get ``saved_bits = 8``; ``nn.GELU`` and
    ``nn.SiLU`` become ``neuzip_amd.nn.FP8Activation``.  Modules whose attribute name
    contains one of ``skip`` (names, or one) are left as they are, and so is what stands below them:
    layers that share their input keep one of 16 bits together, but 8 bits each, so for
    three of them (q, k and v) 16 bits are less.

    A product ``silu(gate) * up`` is no module: its factors are kept as they were, until
    the block calls ``ops.fp8_activation(gate, "silu", up)`` itself."""
    from neuzip_amd.nn import FP8Activation, Linear

    if isinstance(skip, str) and skip:
        skip = (skip,)  # one name, not its letters
    kept = _heads(module, *skip) if skip else set()

    def make(m):
        if isinstance(m, Linear):
            m.saved_bits = 8
        elif isinstance(m, torch.nn.GELU):
            return FP8Activation("gelu" if m.approximate == "none" else "gelu_tanh")
        elif isinstance(m, torch.nn.SiLU):
            return FP8Activation("silu")
        return None

    return _replace(module, prefix, make, {}, kept)
