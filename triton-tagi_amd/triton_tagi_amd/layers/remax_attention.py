"""Causal attention with Remax scores over sequences of any length, trained and served.

Beside MultiheadAttentionV2 (triton_tagi/layers/multihead_attention.py:64-294: no mask, as many
key heads as query heads, no positions, scores kept): queries see the tokens up to their own,
several query heads may share a key head, queries and keys may be normed head by head and turned
by their positions, and no score is stored (``kernels.remax_attention``). As there, projections are
three Linear layers run as one product, heads are read in place from it, and an output projection
is a Linear of the network's own.

Serving keeps the tokens' keys and values in the pages of a cache (``kernels.KVCache``) of float32,
bfloat16 or 8 bits: ``prompt`` runs whole sequences and writes them, ``step`` one token at a time.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch import Tensor

from ..base import LearnableLayer
from ..kernels.common import fused_backward_delta, linear_forward
from ..kernels.kv_cache import KVCache, cache_read, cache_write, new_kv_cache
from ..kernels.remax_attention import remax_attention, remax_attention_backward_into, remax_attention_step
from ..kernels.rotary import qk_norm_rotary, qk_norm_rotary_backward_into, rotary_frequencies
from ..update.parameters import update_parameters_multi
from ._qkv import QkvProjections
from .rms_norm import RMSNorm


@dataclass
class AttentionState:
    """What a RemaxAttention keeps of a batch of sequences: ``lengths`` (B,) int64 tokens of each in
    the pages that ``table`` names. ``used``: no length is above it, as the host counts them; None
    where it does not (a recorded graph's replays advance the lengths), and every call that is not
    recorded reads them back, as it does where the count would not fit and the lengths may."""

    cache: KVCache
    table: Tensor
    lengths: Tensor
    used: int | None = None

    @property
    def room(self) -> int:
        return self.table.shape[1] * self.cache.km.shape[2]

    def clone(self) -> "AttentionState":
        cache = KVCache(*(None if t is None else t.clone() for t in self.cache))
        return AttentionState(cache, self.table, self.lengths.clone(), self.used)


class RemaxAttention(QkvProjections):
    _backward_reads = "_cache"

    def __init__(self, embed_dim: int, num_heads: int, num_kv_heads: int | None = None, max_len: int = 2048,
                 qk_norm: bool = True, rotary: bool = True, rotary_base: float = 10000.0, rotary_sections=None,
                 bias: bool = False, gain_weight: float = 1.0, gain_bias: float = 1.0, init_method: str = "He",
                 cache_dtype: torch.dtype = torch.float32, page_size: int = 64, device: str = "cuda") -> None:
        """``num_kv_heads``: key and value heads, a divisor of ``num_heads``. ``max_len``: tokens of a
        served sequence. ``qk_norm``: RMSNorm of each query and key head. ``rotary``: queries and keys
        turn by their positions, all pairs (u, u + head_dim / 2) of a head; ``rotary_sections`` splits
        the pairs among several axes of positions, which this layer's ``forward`` then takes: a
        ``Sequential`` passes none, and ``prompt`` and ``step`` know only the tokens' order, so they
        refuse such a layer. ``cache_dtype``, ``page_size``: of the cache that serving keeps."""
        num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if embed_dim % num_heads != 0:
            raise ValueError(f"embed_dim ({embed_dim}) must be divisible by num_heads ({num_heads})")
        if num_kv_heads < 1 or num_heads % num_kv_heads != 0:
            raise ValueError(f"num_heads ({num_heads}) must be divisible by num_kv_heads ({num_kv_heads})")
        self.head_dim = embed_dim // num_heads
        if self.head_dim > 128:
            raise ValueError(f"RemaxAttention supports head dimensions up to 128, got {self.head_dim}")
        if rotary and self.head_dim % 2:
            raise ValueError(f"rotary positions need an even head dimension, got {self.head_dim}")
        if max_len < 1 or page_size < 1:
            raise ValueError(f"bad sizes: max_len {max_len}, page_size {page_size}")
        if rotary_sections is not None:
            rotary_sections = tuple(int(n) for n in rotary_sections)
            if not rotary or sum(rotary_sections) != self.head_dim // 2 or min(rotary_sections) < 0:
                raise ValueError(f"rotary_sections: expected counts that add up to {self.head_dim // 2} pairs, got "
                                 f"{rotary_sections}")
        self.embed_dim = embed_dim
        self.num_heads = num_heads
        self.num_kv_heads = num_kv_heads
        self.max_len = max_len
        self.rotary_sections = rotary_sections
        self.has_bias = bias
        self.init_method = init_method
        self.gain_weight = gain_weight
        self.gain_bias = gain_bias
        self.cache_dtype = cache_dtype
        self.page_size = page_size
        self.device = torch.device(device)
        self._make_projections(embed_dim, num_kv_heads * self.head_dim)
        self.q_norm = self.k_norm = None
        if qk_norm:
            self.q_norm = RMSNorm([self.head_dim], device=device)
            self.k_norm = RMSNorm([self.head_dim], device=device)
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self._turns = rotary_frequencies(self.head_dim // 2, rotary_base, device="cpu") if rotary else None
        self._turns_on: dict[torch.device, Tensor] = {}
        self._cache: dict | None = None

    def _norms(self) -> tuple:
        return () if self.q_norm is None else (self.q_norm, self.k_norm)

    def sublayers(self) -> tuple:
        return (*self._projections(), *self._norms())

    @property
    def _learnable(self) -> list:
        """The layers that hold the parameters, in the order in which a checkpoint saves them."""
        return list(self.sublayers())

    # -------------------------------------------------------------------------- forward
    def _frequencies(self, device: torch.device) -> Tensor | None:
        if self._turns is None:
            return None
        t = self._turns_on.get(device)
        if t is None:
            t = self._turns_on[device] = self._turns.to(device)
        return t

    def _rotary(self, device, positions) -> dict:
        """The arguments that the forward and the backward of the norms and turns share."""
        w = None
        if self.q_norm is not None:
            w = (self.q_norm.mw, self.q_norm.Sw, self.k_norm.mw, self.k_norm.Sw)
        if self._turns is None:
            return dict(weights=w)
        return dict(positions=positions, frequencies=self._frequencies(device), weights=w,
                    sections=self.rotary_sections)

    def _project(self, ma: Tensor, Sa: Tensor, positions):
        """What the backward reads, and the six (B, T, heads, D) operands; ``positions`` (B, T)."""
        E, H, G, D = self.embed_dim, self.num_heads, self.num_kv_heads, self.head_dim
        if ma.shape[-1] != E:
            raise ValueError(f"Expected last dim {E}, got {ma.shape[-1]}")
        flat_m = ma.reshape(-1, E).contiguous()
        flat_S = None if Sa is None else Sa.reshape(-1, E).contiguous()
        qkv = self._qkv_params()
        w_m, w_S, b_m, b_S = (qkv.get(a) for a in self._QKV_ATTRS)
        if flat_m.shape[0] == 0:  # no tokens: nothing to project
            out = (torch.empty(0, self._ends[2], device=ma.device),) * 2
        else:
            out = linear_forward(flat_m, flat_S, w_m, w_S, b_m, b_S)
        m, S = (t.view(*ma.shape[:2], H + 2 * G, D) for t in out)
        (mq, mk, mv), (Sq, Sk, Sv) = ((t[:, :, :H], t[:, :, H:H + G], t[:, :, H + G:]) for t in (m, S))
        kept = dict(ma_in=flat_m, w_m=w_m, w_S=w_S, b_S=b_S, raw=(mq, mk), inv=None, rotary=None)
        if self.q_norm is not None or self._turns is not None:
            kept["rotary"] = self._rotary(ma.device, positions)
            eps = self.q_norm.eps if self.q_norm is not None else 0.0
            mq, Sq, mk, Sk, kept["inv"] = qk_norm_rotary(mq, Sq, mk, Sk, eps=eps, **kept["rotary"])
        return kept, (mq, Sq, mk, Sk, mv, Sv)

    def _positions(self, ma: Tensor, starts: Tensor | None, positions: Tensor | None) -> Tensor | None:
        if self._turns is None:
            if positions is not None:
                raise ValueError("positions: this layer has no rotary positions")
            return None
        if positions is None:
            if self.rotary_sections is not None:
                raise ValueError("positions: needed with rotary_sections")
            B, T = ma.shape[:2]
            t = torch.arange(T, device=ma.device)
            return t.expand(B, T) if starts is None else starts[:, None] + t
        return positions

    def forward(self, ma: Tensor, Sa: Tensor, lengths: Tensor | None = None,
                positions: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """(B, S, E) moments to (B, S, E). ``lengths`` (B,): sequences of a padded batch end there;
        their later tokens get zeros and leave no deltas. ``positions`` (B, S) or (B, S, axes): what
        queries and keys turn by; 0, 1, ... without. The mask goes by the tokens' order alone."""
        if ma.dim() != 3:
            raise ValueError(f"RemaxAttention: expected (batch, sequence, features), got {tuple(ma.shape)}")
        kept, ops = self._project(ma, Sa, self._positions(ma, None, positions))
        for p in self._projections():
            p.ma_in, p._input_shape = kept["ma_in"], ma.shape
        mo, So, rows = remax_attention(*ops, scale=self._scale, lengths=lengths, return_rows=True)
        self._cache = dict(kept, ops=ops[:5], rows=rows, lengths=lengths)
        return mo.view(ma.shape), So.view(ma.shape)

    def backward(self, delta_mz: Tensor, delta_Sz: Tensor) -> tuple[Tensor, Tensor]:
        c = self._kept()
        H, G, D, E = self.num_heads, self.num_kv_heads, self.head_dim, self.embed_dim
        shape = c["ops"][0].shape
        B, T = shape[:2]
        # the deltas of Q, K and V side by side, for one projection backward
        dm, dS = (torch.empty(B, T, H + 2 * G, D, device=delta_mz.device, dtype=torch.float32) for _ in range(2))
        q, k, v = ((dm[:, :, a:b], dS[:, :, a:b]) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
        remax_attention_backward_into((*q, *k, *v), *c["ops"], delta_mz.reshape(shape), delta_Sz.reshape(shape),
                                      c["rows"], scale=self._scale, lengths=c["lengths"])
        if c["rotary"] is not None:  # in place: queries and keys as attention read them, then before the norm
            dw = qk_norm_rotary_backward_into((*q, *k), *q, *k, *c["raw"], c["inv"], **c["rotary"])
            if dw:
                n, m = self._norms()
                n.delta_mw, n.delta_Sw, m.delta_mw, m.delta_Sw = dw
        dm, dS = dm.view(B * T, self._ends[2]), dS.view(B * T, self._ends[2])
        self._projection_param_deltas(c, dm, dS)
        dma, dSa = fused_backward_delta(dm, dS, c["w_m"])  # the three projections' sum
        return dma.reshape(B, T, E), dSa.reshape(B, T, E)

    # --------------------------------------------------------------------------- update
    def _update_items(self):
        return super()._update_items() + [it for n in self._norms() for it in n._update_items()]

    def _update_groups(self):
        groups = super()._update_groups()
        if len(groups) > 2:  # the projections' own items: with the norms' already
            return groups
        return groups + [it for n in self._norms() for it in n._update_items()]

    def update(self, cap_factor: float) -> None:
        update_parameters_multi(self._update_groups(), cap_factor)

    @property
    def num_parameters(self) -> int:
        return sum(p.num_parameters for p in self.sublayers() if isinstance(p, LearnableLayer))

    # -------------------------------------------------------------------------- serving
    def new_state(self, batch: int, device=None) -> AttentionState:
        """The state of ``batch`` sequences before their first token, with room for ``max_len`` each."""
        dev = self.device if device is None else torch.device(device)
        width = -(-self.max_len // self.page_size)
        cache = new_kv_cache(batch * width, self.num_kv_heads, self.page_size, self.head_dim, self.cache_dtype, dev)
        table = torch.arange(batch * width, device=dev, dtype=torch.int32).view(batch, width)
        return AttentionState(cache, table, torch.zeros(batch, device=dev, dtype=torch.int64), 0)

    def _bound(self, state: AttentionState, tokens: int, added: Tensor | None = None) -> int:
        """No length is above it after ``tokens`` more (of each sequence ``added`` (B,) where given), which
        the room has to hold. The host counts every sequence as if it took all ``tokens``; where that
        count does not fit, or there is none, the lengths are read back. A recorded call keeps the
        whole room: every replay finds other lengths (and ``added``), which are its caller's to bound."""
        recorded = torch.cuda.is_current_stream_capturing()
        limit = min(self.max_len, state.room)
        most = None if state.used is None or (recorded and added is not None) else state.used + tokens
        if not recorded and (most is None or most > limit):
            most = int((state.lengths + (tokens if added is None else added)).max())
        if most is not None and most > limit:
            raise ValueError(f"RemaxAttention: a sequence of up to {most} tokens, max_len is {limit}")
        return state.room if recorded else most

    def prompt(self, ma: Tensor, Sa: Tensor, lengths: Tensor | None = None, state: AttentionState | None = None):
        """``forward`` after the tokens of ``state`` (none without) that keeps nothing for a backward:
        (mo, So, the state with these tokens); ``state`` is copied, not written. A fresh prompt's own
        tokens are seen unrounded, earlier ones as the cache holds them."""
        if ma.dim() != 3:
            raise ValueError(f"RemaxAttention: expected (batch, sequence, features), got {tuple(ma.shape)}")
        B, T = ma.shape[:2]
        fresh = state is None
        if not fresh and (not isinstance(state, AttentionState) or state.lengths.shape[0] != B):
            raise ValueError(f"state: expected an AttentionState of {B} sequences")
        if fresh:
            state = self.new_state(B, ma.device)
        added = torch.full_like(state.lengths, T) if lengths is None else lengths.clamp(0, T).to(torch.int64)
        if tuple(added.shape) != (B,):
            raise ValueError(f"lengths: expected ({B},), got {tuple(added.shape)}")
        bound = self._bound(state, T, None if lengths is None else added)
        end = state if fresh else state.clone()
        starts = None if fresh else end.lengths
        _, ops = self._project(ma, Sa, self._positions(ma, starts, None))
        cache_write(end.cache, *ops[2:], end.table, starts, added)
        total = end.lengths + added
        keys = ops[2:] if fresh else cache_read(end.cache, end.table, total, bound)
        mo, So = remax_attention(*ops[:2], *keys, scale=self._scale, lengths=total, starts=starts)
        end.lengths, end.used = total, None if torch.cuda.is_current_stream_capturing() else bound
        return mo.view(ma.shape), So.view(ma.shape), end

    def _check_state(self, state, batch: int, active: Tensor | None) -> None:
        if not isinstance(state, AttentionState) or state.lengths.shape[0] != batch:
            raise ValueError(f"state: expected an AttentionState of {batch} sequences")
        if active is not None and (active.dtype not in (torch.bool, torch.uint8) or tuple(active.shape) != (batch,)):
            raise TypeError(f"active: expected a bool or uint8 tensor of ({batch},)")

    def check_step(self, state: AttentionState, batch: int, active: Tensor | None = None) -> None:
        """Refuses what ``step`` would refuse of a state, before any layer of a network has taken the token."""
        self._check_state(state, batch, active)
        if state.used is None or state.used >= min(self.max_len, state.room):  # else the count says enough
            self._bound(state, 1, None if active is None else (active != 0).to(torch.int64))

    def step(self, ma: Tensor, Sa: Tensor, state: AttentionState, active: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """One token of every sequence, (B, E) or (B, 1, E); ``state`` is advanced in place. ``active``
        (B,): sequences that are off keep their state and get zeros. A recorded graph's replays
        advance the state without the host: at most ``max_len`` tokens are its caller's to keep, and
        calls on this state that are not recorded read its lengths back (a wait for the GPU)."""
        if ma.dim() not in (2, 3) or (ma.dim() == 3 and ma.shape[1] != 1):
            raise ValueError(f"RemaxAttention.step: expected (batch, features) or (batch, 1, features), "
                             f"got {tuple(ma.shape)}")
        B, E = ma.shape[0], ma.shape[-1]
        self._check_state(state, B, active)
        on = None if active is None else (active != 0).to(torch.int64)
        bound = self._bound(state, 1, on)
        at = state.lengths
        positions = self._positions(ma.reshape(B, 1, E), at, None)
        _, ops = self._project(ma.reshape(B, 1, E), None if Sa is None else Sa.reshape(B, 1, E), positions)
        cache_write(state.cache, *ops[2:], state.table, at, on)
        at.add_(1 if on is None else on)
        seen = at if on is None else at * on
        if torch.cuda.is_current_stream_capturing():
            state.used = None
        elif state.used is not None:
            state.used = bound
        most = -(-bound // 256) * 256
        mo, So = remax_attention_step(ops[0][:, 0], ops[1][:, 0], state.cache, state.table, seen, scale=self._scale,
                                      max_len=most)
        return mo.view(ma.shape), So.view(ma.shape)

    def __repr__(self) -> str:
        return (f"RemaxAttention(embed_dim={self.embed_dim}, num_heads={self.num_heads}, "
                f"num_kv_heads={self.num_kv_heads}, bias={self.has_bias})")
