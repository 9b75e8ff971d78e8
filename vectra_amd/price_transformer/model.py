"""The price Transformer.

The subject property and its K comparables become K + 1 tokens; pre-norm
Transformer blocks with spatial (RBF) attention mix them, and the subject
token is read out as a correction to the comparables' mean log price.  Same
architecture and forward semantics as the reference's
models/price_transformer/model.py:39-282; trimming comparables to the search
radius (with a nearest-neighbour fallback) is branch-free tensor code, so
TorchDynamo captures the forward pass as a single graph, every attention
site stays visible to the rewrite, and a forward pass never waits for the
GPU.
"""

import dataclasses
import math
import typing
from collections.abc import Mapping

import torch
from torch import nn

from vectra_amd.price_transformer import candidate_encoder
from vectra_amd.price_transformer import microhood
from vectra_amd.price_transformer import plain_modules
from vectra_amd.price_transformer import spatial_attention


@dataclasses.dataclass(frozen=True)
class ModelConfig:
    embedding_dim: int = 128
    attribute_dim: int = 5
    d_model: int = 128
    num_heads: int = 4
    num_layers: int = 2
    ffn_dim: int = 256
    num_candidates: int = 64
    min_candidates: int = 4  # kept when no comparable lies inside the radius
    ffn_gate: bool = False  # a gated (SiLU) feed-forward block; no counterpart in the reference
    # Of each branch's output before the residual, in training; no counterpart in the reference.
    dropout: float = 0.0

    @classmethod
    def from_dict(cls, values: Mapping[str, typing.Any]) -> 'ModelConfig':
        names = {f.name for f in dataclasses.fields(cls)}
        return cls(**{k: v for k, v in values.items() if k in names})

    def to_dict(self) -> dict[str, typing.Any]:
        """The fields as the reference writes them; `ffn_gate` and `dropout` only where
        they are set."""
        values = dataclasses.asdict(self)
        for own in ('ffn_gate', 'dropout'):
            if not values[own]:
                del values[own]
        return values


class PricingInputs(typing.NamedTuple):
    """One batch of requests, in forward-argument order."""

    query_embedding: torch.Tensor  # [B, E]
    query_attributes: torch.Tensor  # [B, A]
    query_location: torch.Tensor  # [B, 2] lat, lon degrees
    query_cell6: torch.Tensor  # [B] int64
    valuation_day: torch.Tensor  # [B] days since epoch
    radius_km: torch.Tensor  # [B]
    cand_embedding: torch.Tensor  # [B, K, E]
    cand_attributes: torch.Tensor  # [B, K, A]
    cand_log_price: torch.Tensor  # [B, K]
    cand_sale_day: torch.Tensor  # [B, K]
    cand_location: torch.Tensor  # [B, K, 2]
    cand_cell6: torch.Tensor  # [B, K] int64
    cand_valid: torch.Tensor  # [B, K] bool

    def to(self, device) -> 'PricingInputs':
        return PricingInputs(*(t.to(device) for t in self))  # pylint: disable=not-an-iterable


def trim_to_radius(distance_km, radius_km, valid, min_keep: int) -> torch.Tensor:
    """Comparables inside the radius; rows with none keep their `min_keep` nearest.

    The reference (models/price_transformer/model.py:96-138) picks between an
    inside-only branch and this nearest-neighbour fallback with a torch.cond
    on "every row has a comparable inside".  Both give the same mask on every
    row the inside-only branch covers, so here the fallback is always taken
    and selected per row: the same mask with no data-dependent branch.  The
    cond's predicate is a device-to-host read on every forward pass, which
    stalls the host until the GPU has caught up, so the model could not be
    launched ahead of the GPU, overlapped with the next batch's copy, or
    captured in a HIP graph.
    """
    inside = valid & (distance_km <= radius_km.unsqueeze(-1))
    nearest = distance_km.masked_fill(~valid, float('inf')).topk(min_keep, dim=-1, largest=False).indices
    fallback = torch.zeros_like(valid).scatter(-1, nearest, True) & valid
    return torch.where(inside.any(-1, keepdim=True), inside, fallback)


class GatedFeedForward(nn.Module):
    """down(silu(gate(x)) * up(x)); the gate's and the up projection's rows lie
    in one weight, as torch.ops.vectra.gated_linear takes them."""

    def __init__(self, d_model: int, hidden: int):
        super().__init__()
        self.gate_up = nn.Linear(d_model, 2 * hidden)
        self.down = nn.Linear(hidden, d_model)

    def forward(self, x):
        gate, up = self.gate_up(x).chunk(2, dim=-1)
        return self.down(nn.functional.silu(gate) * up)


class Block(nn.Module):
    """Pre-norm Transformer block with spatial attention."""

    dense_checkpoint: str | None = None  # as SpatialAttention's
    norm_kernels = False  # residual sums and norms on torch.ops.vectra.residual_norm
    dropout = 0.0
    index = 0  # of the block: its two branches draw as streams 2 index and 2 index + 1

    def __init__(self, config: ModelConfig, index: int = 0):
        super().__init__()
        self.dropout, self.index = config.dropout, index
        self.norm1 = nn.LayerNorm(config.d_model)
        self.attention = spatial_attention.SpatialAttention(config.d_model, config.num_heads)
        self.norm2 = nn.LayerNorm(config.d_model)
        if config.ffn_gate:
            self.ffn = GatedFeedForward(config.d_model, config.ffn_dim)
        else:
            self.ffn = nn.Sequential(
                nn.Linear(config.d_model, config.ffn_dim),
                nn.GELU(),
                nn.Linear(config.ffn_dim, config.d_model),
            )

    def forward(self, x, key_bias, rng=None, normed=None, following=None):
        """x [B, N, d_model] through both branches.  rng: what dropout draws from (None:
        none is dropped).  normed: norm1(x), where the caller has it.  following: a norm
        of the result, which is returned beside it then."""
        if not self.training:
            rng = None
        if normed is None:
            normed = self.norm1(x)
        joined = self.norm_kernels and plain_modules.is_plain_norm(self.norm2, x.shape[-1])
        if (self.dense_checkpoint is not None and rng is None and not joined
                and plain_modules.is_plain(self.attention, spatial_attention.SpatialAttention)):
            x = self.attention(normed, key_bias, residual=x)
            normed = self.norm2(x)
        else:
            x, normed = self._join(self.attention(normed, key_bias), x, self.norm2, rng, 2 * self.index)
        if self.dense_checkpoint is None:
            branch = self.ffn(normed)
        elif rng is None and following is None:
            return self._feed_forward(normed, x, self.dense_checkpoint)
        else:
            branch = self._feed_forward(normed, None, self.dense_checkpoint)
        if following is None:
            return x + self._drop(branch, rng, 2 * self.index + 1)
        return self._join(branch, x, following, rng, 2 * self.index + 1)

    def _drop(self, branch, rng, stream):
        return branch if rng is None else torch.ops.vectra.dropout(branch, self.dropout, rng, stream)

    def _join(self, branch, x, norm, rng, stream):
        """The residual stream with a branch's output, and `norm` of it: in one pass
        where the norm is a plain one and the types are the operator's (under autocast
        branches may be narrower than the stream, never wider)."""
        if (self.norm_kernels and plain_modules.is_plain_norm(norm, x.shape[-1])
                and x.dtype in (branch.dtype, torch.float32)
                and (norm.weight is None or norm.weight.dtype in (branch.dtype, torch.float32))):
            return torch.ops.vectra.residual_norm(branch, x, norm.weight, norm.bias, norm='layer', eps=norm.eps,
                                                  p=0.0 if rng is None else self.dropout, rng=rng, stream=stream)
        x = x + self._drop(branch, rng, stream)
        return x, norm(x)

    def _feed_forward(self, x, residual, checkpoint):
        """The feed-forward block on the dense operators, onto the residual if there is one."""
        ffn = self.ffn
        if (plain_modules.is_plain(ffn, GatedFeedForward) and plain_modules.is_plain(ffn.gate_up, nn.Linear)
                and plain_modules.is_plain(ffn.down, nn.Linear)):
            first, second = ffn.gate_up, ffn.down
            hidden = torch.ops.vectra.gated_linear(x, first.weight, first.bias, 'silu', checkpoint)
        elif plain_modules.is_plain_mlp(ffn):
            first, second = ffn[0], ffn[2]
            hidden = torch.ops.vectra.linear(x, first.weight, first.bias, None, 'gelu', checkpoint)
        else:
            return ffn(x) if residual is None else residual + ffn(x)
        return torch.ops.vectra.linear(hidden, second.weight, second.bias, residual, 'none', checkpoint)


class PriceTransformer(nn.Module):
    def __init__(self, config: ModelConfig):
        super().__init__()
        self.config = config
        self.query_encoder = candidate_encoder.QueryEncoder(
            config.embedding_dim, config.attribute_dim, config.d_model
        )
        self.candidate_encoder = candidate_encoder.CandidateEncoder(
            config.embedding_dim, config.attribute_dim, config.d_model
        )
        self.blocks = nn.ModuleList([Block(config, i) for i in range(config.num_layers)])
        self.norm = nn.LayerNorm(config.d_model)
        self.head = nn.Linear(config.d_model, 1)
        self._block_dtype = torch.float32
        if config.dropout:
            if not 0.0 <= config.dropout < 1.0 - 2 ** -17:  # (in steps of 2^-16)
                raise ValueError(f'dropout must be at least 0 and at most 1 - 2^-16, not {config.dropout}')
            # The seed of dropout's generator and the number of training passes so far.
            # Part of a training run, not of the weights, and of this process's run: no
            # buffer, which data parallel wrappers would overwrite with the first rank's.
            self.dropout_rng = torch.tensor([torch.initial_seed() % 2**63, 0], device='cpu')

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        if self.config.dropout:
            self._move_dropout(fn(self.dropout_rng).device)
        return self

    def _move_dropout(self, device):
        """The state goes where the weights go, but not where it would be lost."""
        if self.dropout_rng.device != device and device.type != 'meta':
            self.dropout_rng = self.dropout_rng.to(device)

    def seed_dropout(self, seed: int, passes: int = 0) -> 'PriceTransformer':
        """Dropout's generator: training pass number `passes` of `seed` comes next.  (Data
        parallel ranks with equal seeds drop the same elements of their batches: each
        gives its own, after wrapping or before.)"""
        if not self.config.dropout:
            raise ValueError('the model has no dropout')
        self.dropout_rng.copy_(torch.tensor([seed, passes]))
        return self

    def dropout_pass(self):
        """What the next pass's dropout draws from, counted on; None where nothing is
        dropped (blocks drop where they are in training, each by itself).  A pass that is
        run again in the backward one (activation checkpointing of the whole model) takes
        it as an argument:

            checkpoint(model, *inputs, model.dropout_pass(), use_reentrant=False)
        """
        if not self.config.dropout or not any(block.training for block in self.blocks):
            return None
        from vectra_amd.kernels import block  # pylint: disable=import-outside-toplevel

        # A copy: the backward pass draws from it again, after later passes too.  Counted
        # on the device, so that each replay of a captured pass draws anew.
        return block.dropout_pass(self.dropout_rng)

    def set_block_dtype(self, dtype: torch.dtype) -> 'PriceTransformer':
        """Runs the Transformer blocks in `dtype`; encoders, geometry and the
        read-out stay fp32 (coordinates in half precision would lose km)."""
        self.blocks.to(dtype)
        self._block_dtype = dtype
        return self

    def set_dense_kernels(self, enabled: bool = True, checkpoint: str = 'none') -> 'PriceTransformer':
        """Runs the linear layers of the blocks and encoders through
        torch.ops.vectra.linear and gated_linear: bias, activation and residual
        in the product's epilogue, for training with the operators' own
        gradients.  `checkpoint='e4m3'`: the blocks keep their layers' inputs
        in 8 bits for the backward pass (the encoders' inputs, prices and
        distances, stay as they are).  The parameters are the same either way.
        Layers that carry hooks, and ones that were wrapped or replaced, are
        called as they are (plain_modules.py)."""
        if enabled:
            from vectra_amd.kernels import dense  # pylint: disable=import-outside-toplevel

            if checkpoint not in dense.CHECKPOINTS:
                raise ValueError(f'checkpoint must be one of {dense.CHECKPOINTS}, not {checkpoint!r}')
        for module in self.modules():  # (those inside wrappers too)
            if isinstance(module, (Block, spatial_attention.SpatialAttention)):
                module.dense_checkpoint = checkpoint if enabled else None
            elif isinstance(module, (candidate_encoder.QueryEncoder, candidate_encoder.CandidateEncoder)):
                module.dense_kernels = enabled
        return self

    def set_norm_kernels(self, enabled: bool = True) -> 'PriceTransformer':
        """Runs the blocks' residual sums and the norms that follow them, dropout
        between them included, through torch.ops.vectra.residual_norm: one pass over
        the tokens each, forward and backward, also across blocks.  For eager runs and
        training: torch.compile fuses them by itself.  With set_dense_kernels the
        residual is added there and not in the products' epilogues.  Norms and blocks
        that carry hooks, and ones that were wrapped or replaced, are called as they
        are."""
        if enabled:
            from vectra_amd.kernels import block  # pylint: disable=import-outside-toplevel

            if self.config.d_model > block.NORM_WIDTH:
                raise ValueError(f'd_model {self.config.d_model} exceeds the widest row of a norm, {block.NORM_WIDTH}')
        for module in self.modules():  # (those inside wrappers too)
            if isinstance(module, Block):
                module.norm_kernels = enabled
        return self

    def _following(self, i: int):
        """The norm that block i computes with its result: the next block's first, where
        calls of the two would do nothing besides."""
        block = self.blocks[i]
        if i + 1 == len(self.blocks) or not plain_modules.is_plain(block, Block) or not block.norm_kernels:
            return None
        after = self.blocks[i + 1]
        plain = plain_modules.is_plain(after, Block) and plain_modules.is_plain_norm(after.norm1, self.config.d_model)
        return after.norm1 if plain else None

    def forward(self, query_embedding, query_attributes, query_location, query_cell6,
                valuation_day, radius_km, cand_embedding, cand_attributes, cand_log_price,
                cand_sale_day, cand_location, cand_cell6, cand_valid, rng=None) -> torch.Tensor:
        """Predicted natural-log prices [B].  rng: this pass's dropout_pass(), where the
        caller has taken it."""
        distance = microhood.haversine_km(query_location, cand_location)
        valid = trim_to_radius(
            distance, radius_km, cand_valid, min(self.config.min_candidates, cand_valid.shape[-1])
        )
        candidates = self.candidate_encoder(
            cand_embedding,
            cand_attributes,
            cand_log_price,
            valuation_day.unsqueeze(-1) - cand_sale_day,
            microhood.relative_offsets_km(query_location, cand_location),
            distance,
            radius_km,
            microhood.same_cell_flags(query_cell6, cand_cell6),
        )
        query = self.query_encoder(query_embedding, query_attributes)
        tokens = torch.cat([query.unsqueeze(1), candidates], dim=1).to(self._block_dtype)
        token_valid = torch.cat([torch.ones_like(valid[:, :1]), valid], dim=1)
        key_bias = torch.zeros_like(token_valid, dtype=tokens.dtype).masked_fill(
            ~token_valid, float('-inf')
        )[:, None, None, :]
        if not self.config.dropout:
            rng = None
        elif rng is None:
            self._move_dropout(tokens.device)  # (where a wrapper has moved the weights one by one)
            rng = self.dropout_pass()
        normed = None
        for i, block in enumerate(self.blocks):
            following = self._following(i)
            if following is not None:
                tokens, normed = block(tokens, key_bias, rng, normed, following)
            elif normed is not None:
                tokens, normed = block(tokens, key_bias, rng, normed), None
            else:  # (a wrapped block need not take more)
                tokens = block(tokens, key_bias) if rng is None or not block.training else block(tokens, key_bias, rng)
        weights = valid.to(cand_log_price.dtype)
        baseline = (cand_log_price * weights).sum(-1) / weights.sum(-1).clamp_min(1.0)
        readout = self.head(self.norm(tokens[:, 0].float()))
        return baseline + readout.squeeze(-1)


def example_inputs(config: ModelConfig, batch_size: int, device='cpu', seed: int = 0) -> PricingInputs:
    """Random inputs of the serving shape around one city (reference model.py:247-282):
    comparables within ~2 km of the subject, the last K/8 of them padding."""
    gen = torch.Generator().manual_seed(seed)
    k = config.num_candidates

    def randn(*shape):
        return torch.randn(*shape, generator=gen)

    center = torch.tensor([37.7749, -122.4194])
    query_location = center + 0.02 * randn(batch_size, 2)
    cand_location = query_location[:, None, :] + 0.02 * randn(batch_size, k, 2)
    cells = torch.randint(0, 1 << 30, (batch_size,), generator=gen)
    valid = torch.ones(batch_size, k, dtype=torch.bool)
    valid[:, k - k // 8 :] = False
    return PricingInputs(
        query_embedding=torch.tanh(randn(batch_size, config.embedding_dim)),
        query_attributes=randn(batch_size, config.attribute_dim),
        query_location=query_location,
        query_cell6=cells,
        valuation_day=torch.full((batch_size,), 20000.0),
        radius_km=torch.full((batch_size,), 5.0),
        cand_embedding=torch.tanh(randn(batch_size, k, config.embedding_dim)),
        cand_attributes=randn(batch_size, k, config.attribute_dim),
        cand_log_price=13.0 + 0.5 * randn(batch_size, k),
        cand_sale_day=20000.0 - 900.0 * randn(batch_size, k).abs(),
        cand_location=cand_location,
        cand_cell6=cells[:, None] + torch.randint(0, 3, (batch_size, k), generator=gen),
        cand_valid=valid,
    ).to(device)


def box_inputs(config: ModelConfig, batch_size: int, device='cpu', seed: int = 0,
               box_km: float = 50.0, max_age_days: float = 730.0) -> PricingInputs:
    """Inputs of the full-model benchmark configuration: attributes ~ N(0, 1),
    subjects and comparables uniform over a `box_km` square, sale dates
    uniform over the `max_age_days` before valuation, embeddings tanh(N(0,1)),
    every comparable valid and a radius covering the box."""
    gen = torch.Generator().manual_seed(seed)
    k = config.num_candidates
    south_west = torch.tensor([37.55, -122.55])
    deg_lat = box_km / (microhood.EARTH_RADIUS_KM * math.pi / 180.0)
    deg_lon = deg_lat / math.cos(math.radians(float(south_west[0]) + deg_lat / 2))
    span = torch.tensor([deg_lat, deg_lon])

    def uniform(*shape):
        return torch.rand(*shape, generator=gen)

    query_location = south_west + span * uniform(batch_size, 2)
    cand_location = south_west + span * uniform(batch_size, k, 2)
    cells = torch.randint(0, 1 << 30, (batch_size,), generator=gen)
    valuation = torch.full((batch_size,), 20000.0)
    return PricingInputs(
        query_embedding=torch.tanh(torch.randn(batch_size, config.embedding_dim, generator=gen)),
        query_attributes=torch.randn(batch_size, config.attribute_dim, generator=gen),
        query_location=query_location,
        query_cell6=cells,
        valuation_day=valuation,
        radius_km=torch.full((batch_size,), box_km * math.sqrt(2.0)),
        cand_embedding=torch.tanh(torch.randn(batch_size, k, config.embedding_dim, generator=gen)),
        cand_attributes=torch.randn(batch_size, k, config.attribute_dim, generator=gen),
        cand_log_price=13.0 + 0.5 * torch.randn(batch_size, k, generator=gen),
        cand_sale_day=valuation[:, None] - max_age_days * uniform(batch_size, k),
        cand_location=cand_location,
        cand_cell6=cells[:, None] + torch.randint(0, 3, (batch_size, k), generator=gen),
        cand_valid=torch.ones(batch_size, k, dtype=torch.bool),
    ).to(device)
