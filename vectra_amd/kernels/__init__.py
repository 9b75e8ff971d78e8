"""The fused RBF-attention operator and a block's dense operators on MI355X.

Importing vectra_amd.kernels (or vectra_amd.kernels.custom_ops) loads the
native libraries and registers torch.ops.vectra.rbf_attention, as importing
vectra_kernels.custom_ops does in the reference
(kernels/vectra_kernels/__init__.py:17).  The dense operators
(torch.ops.vectra.linear and its relatives) are registered with it.
"""

from vectra_amd.kernels import block  # noqa: F401  (registers the fakes of what stands between them)
from vectra_amd.kernels import custom_ops  # noqa: F401  (registers the op)
from vectra_amd.kernels import dense  # noqa: F401  (registers the dense operators' fakes)
