"""Which modules an operator may stand in for.

PriceTransformer.set_dense_kernels and set_norm_kernels read the parameters of
linear layers and norms instead of calling them.  That is the same function only where a call of the module
would do nothing else: for a module of the expected class itself (a subclass, a
wrapper or a parametrised layer has a forward of its own) that carries no hooks.
"""

import torch
from torch import nn


def is_plain(module: nn.Module, kind: type) -> bool:
    """Whether calling `module` runs `kind`'s forward and nothing besides."""
    return (type(module) is kind and 'forward' not in module.__dict__
            and not (module._forward_hooks or module._forward_pre_hooks  # pylint: disable=protected-access
                     or module._backward_hooks or module._backward_pre_hooks)
            and not torch.nn.modules.module._has_any_global_hook())  # pylint: disable=protected-access


def is_plain_mlp(module: nn.Module) -> bool:
    """Whether `module` is a plain Linear - GELU - Linear sequence."""
    if not is_plain(module, nn.Sequential) or len(module) != 3:
        return False
    first, act, second = module
    return (is_plain(first, nn.Linear) and is_plain(act, nn.GELU) and act.approximate == 'none'
            and is_plain(second, nn.Linear))


def is_plain_norm(module: nn.Module, width: int) -> bool:
    """Whether `module` is a plain layer norm over rows of `width`."""
    return is_plain(module, nn.LayerNorm) and tuple(module.normalized_shape) == (width,)
