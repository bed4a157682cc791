"""Python surface of the hybrid extension (csrc/gdn_rows.cu, gdn_chunk.cu, rope_part.cu, attn_shared.cu): the blocks of the Gated-DeltaNet
family where a step has more than one new row per sequence, its softmax blocks, and attention of batches behind a shared prefix.

As in :mod:`llaminar_b200.ops`, every call launches hand-written CUDA on the current stream; there is no fallback.  Arguments are checked
on the host, indices that lie on the device (slots, page ids, row ranges) are the caller's promise.  The PyTorch form of the
recurrence is in :mod:`llaminar_b200.models.gdn`.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _count, scratch_for
from . import build as _build


_ready = False


def ext():
    global _ready
    mod = _build.load(_build.HYBRID)
    if not _ready:
        from ..utils.env import debug_env
        mod.set_pdl(bool(debug_env().pdl))
        _ready = True
    return mod


GDN_HEAD_SIZES = (32, 64, 128)
SHARED_HEAD_SIZES = (64, 128, 256)     # of rope_part_kv and attn_decode_shared
GDN_CHUNK = 64                 # rows of a chunk
# Rows from which the chunk form is taken, for the call and per sequence.  16 / 32 heads, row by row against chunks: 1 sequence of 16 rows 23 / 32 us, of 37 rows
# 46 / 31; 8 of 8 rows 33 / 53; 32 of 8 rows 99 / 171, of 24 rows 220 / 172.  Lengths lie on the device: if all but one sequence have a row each, the long one costs
# 1 us a row, which the bound per sequence keeps below twice the time in chunks.
GDN_CHUNK_MIN_ROWS = (16, 9)
GDN_WORKSPACE = 256 << 20      # bytes that a pass of the chunk form may hold; longer prompts take several passes


def _gdn_workspace(inp: torch.Tensor, n_seqs: int, n_k: int, n_v: int, d: int):
    """Workspace of the chunk form, or None where the rows go one after the other."""
    if d != 128 or n_seqs == 0 or inp.shape[0] < GDN_CHUNK_MIN_ROWS[0] + GDN_CHUNK_MIN_ROWS[1] * n_seqs:
        return None
    one = ext().gdn_chunk_bytes(1, n_k, n_v)
    units = max(1, min(inp.shape[0] // GDN_CHUNK + n_seqs, GDN_WORKSPACE // one))
    return torch.empty(units * one + 1024, dtype=torch.uint8, device=inp.device)


def gdn_prefill(inp: torch.Tensor, C: int, z_off: int, ab_off: int, conv_w: torch.Tensor, ssm_a: torch.Tensor, dt_bias: torch.Tensor,
                norm_w: torch.Tensor, conv_state: torch.Tensor, rec: torch.Tensor, positions: torch.Tensor, cu: torch.Tensor,
                slots: torch.Tensor, out: torch.Tensor, n_k: int, v_head_offset: int, eps: float) -> None:
    """A Gated-DeltaNet block between its input and output projections for the new rows of a packed batch (arguments as in `gdn_step`).
    Rows cu[b] .. cu[b + 1] of ``inp`` and ``out`` are sequence b's; its state, the slot slots[b] of the layer's fp32 pools conv_state
    [slots, C, K - 1] and rec [slots, n_v, d, d], is advanced in place.  A sequence whose first row has position 0 starts from zeros, whatever
    its slot holds.  Sequences have slots of their own; one without rows keeps its state, and rows outside of all sequences are left as
    they are.  d is 32, 64 or 128; ssm_a is not positive, so that no decay grows.  Values of a row that are not finite reach no row in front of it, no other sequence
    and no head that does not read them; in chunks all outputs of a head behind such a key, value or gate are NaN, and its state."""
    ws = _gdn_workspace(inp, slots.numel(), n_k, rec.shape[1], rec.shape[-1]) if inp.is_cuda else None
    _count(ext().gdn_prefill(inp, C, z_off, ab_off, conv_w, ssm_a, dt_bias, norm_w, conv_state, rec, positions, cu, slots, out, n_k, v_head_offset, eps,
                             ws, scratch_for(inp.device).status if ws is not None else None))


@dataclass
class GdnStash:
    """What `gdn_verify` keeps for `gdn_commit`: decay, key and correction of every row and head, the convolution's inputs, and the sequences' slots (the tensor itself:
    it still says the same at the commit)."""
    decay: torch.Tensor            # [B, R, n_v]
    key: torch.Tensor              # [B, R, n_v, d]
    correction: torch.Tensor       # [B, R, n_v, d]
    inputs: torch.Tensor           # [B, R, C] bf16
    slots: torch.Tensor            # [B]
    n_k: int


def gdn_verify(inp: torch.Tensor, C: int, z_off: int, ab_off: int, conv_w: torch.Tensor, ssm_a: torch.Tensor, dt_bias: torch.Tensor,
               norm_w: torch.Tensor, conv_state: torch.Tensor, rec: torch.Tensor, slots: torch.Tensor, out: torch.Tensor, n_k: int,
               v_head_offset: int, eps: float) -> GdnStash:
    """The same for R drafted rows of every sequence (``inp`` [B * R, ...]) with the state left alone: the outputs are those of feeding
    the rows one by one, and `gdn_commit` advances the states once it is known how many of them are accepted."""
    B = slots.numel()
    if B == 0 or inp.shape[0] % B:
        raise ValueError(f"{inp.shape[0]} rows cannot be shared out evenly between {B} sequences")
    R, n_v, d = inp.shape[0] // B, rec.shape[1], rec.shape[2]
    f = lambda *s: torch.empty(*s, dtype=torch.float32, device=inp.device)
    st = GdnStash(f(B, R, n_v), f(B, R, n_v, d), f(B, R, n_v, d), torch.empty(B, R, C, dtype=torch.bfloat16, device=inp.device), slots, n_k)
    _count(ext().gdn_verify(inp, C, z_off, ab_off, conv_w, ssm_a, dt_bias, norm_w, conv_state, rec, slots, out, n_k, v_head_offset, eps,
                            [st.decay, st.key, st.correction, st.inputs], scratch_for(inp.device).status))
    return st


def gdn_commit(stash: GdnStash, n_rows: torch.Tensor, conv_state: torch.Tensor, rec: torch.Tensor) -> None:
    """Advance the state of every sequence of ``stash`` by its first n_rows[b] rows (int32 on the device; 0 leaves it as it is)."""
    ext().gdn_commit([stash.decay, stash.key, stash.correction, stash.inputs], n_rows, conv_state, rec, stash.slots, stash.n_k)
    _count()


def rope_part_kv(rows: torch.Tensor, q_out: torch.Tensor, kv: torch.Tensor, q_norm: torch.Tensor | None, k_norm: torch.Tensor | None, freqs: torch.Tensor,
                 magnitude: float, positions: torch.Tensor, seq_ids: torch.Tensor, block_table: torch.Tensor, n_heads: int, n_kv_heads: int,
                 head_dim: int, eps: float, *, gated: bool = False, interleaved: bool = False) -> None:
    """Projected rows [query per head | keys | values], with ``gated`` [(query, gate) per head | keys | values] -> queries q_out [tokens, heads, head size] and the
    tokens' entries of the paged cache ``kv`` (bf16, or 8-bit as in `rope_kv`).  Queries and keys are RMS-normed per head (gains of a head, or None: as they
    are), then the first 2 len(freqs) values turn by position x freqs (float64, on the device; `Rotary.frequencies` has them for plain and
    scaled rotations), pairs (i, i + len(freqs)) or, ``interleaved``, (2i, 2i + 1), times ``magnitude``; the rest passes.  Head sizes 64, 128 and 256;
    positions are not negative and their page is in block_table[seq_ids[t]]."""
    ext().rope_part_kv(rows, q_out, kv, q_norm, k_norm, freqs, float(magnitude), positions, seq_ids, block_table, n_heads, n_kv_heads, head_dim, eps,
                       bool(gated), bool(interleaved))
    _count()


def attn_decode_shared(q: torch.Tensor, kv: torch.Tensor, out: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, shared_len: torch.Tensor,
                       n_heads: int, n_kv_heads: int, head_dim: int, rows_per_seq: int, scale: float, scratch, *, gate: torch.Tensor | None = None,
                       max_shared: int, max_tail: int = 0, prefix_row: int = 0) -> None:
    """`attn_decode` over bf16 pages for sequences that share their first keys, which are read and multiplied once for all of them: keys 0 .. shared_len (one
    int32 on the device), in the pages that block_table[prefix_row] begins with.  Those pages, the last one whole even if the prefix ends in it, stand
    in front of the table of every sequence whose rows all see the prefix; a shorter sequence, or one of no keys, takes nothing from it.  ``max_shared``
    (host; 0: nothing is shared) and ``max_tail`` (most keys of a sequence behind the prefix; 0: unknown) only decide how the keys are shared out.
    ``gate`` [rows, heads, head size]: its sigmoid multiplies the result.  ``scale`` is positive.  Head sizes 64, 128 and 256, up to 16 rows x query heads per K/V head."""
    _count(ext().attn_decode_shared(q, kv, out, block_table, seq_lens, shared_len, n_heads, n_kv_heads, head_dim, rows_per_seq, scale, gate, max_shared, max_tail,
                                    prefix_row, scratch.attn_tickets, scratch.status))


def bounds_status(reset: bool = True) -> int:
    return int(ext().bounds_status(bool(reset)))
