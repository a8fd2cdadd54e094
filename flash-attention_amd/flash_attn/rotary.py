"""Rotary position embeddings used by FlashMHA(use_rotary_emb=...), interface-compatible with the reference's
flash_attn/rotary.py (:22-135).  The general functions are PyTorch elementwise ops as in the reference; for the case
the attention modules use, q and k of a packed (batch, seqlen, 3, nheads, headdim) GPU tensor, `apply_rotary_emb_qkv_`
rotates both in place in one pass of a HIP kernel (fa_rotary), with a matching backward.

Convention (rotary.py:22-42,66-87): channel pairs are interleaved, (x[2i], x[2i+1]) is rotated by angle
pos * 10000^(-2i/dim):   x'[2i] = x[2i] cos - x[2i+1] sin,   x'[2i+1] = x[2i+1] cos + x[2i] sin.
The cos/sin tables are rounded to the input dtype before use, as the reference does.
"""
import math
from typing import Tuple

import torch


def rotate_half(x):
    """(x0, x1, x2, x3, ...) -> (-x1, x0, -x3, x2, ...)"""
    pairs = x.reshape(*x.shape[:-1], -1, 2)
    return torch.stack((-pairs[..., 1], pairs[..., 0]), dim=-1).reshape(x.shape)


def apply_rotary_pos_emb(x, cos, sin, seq_dimension: int = -2):
    """x: (..., s, d) if seq_dimension == -2, (..., s, h, d) if -3.  cos, sin: (>= s, d)."""
    n = x.shape[seq_dimension]
    cos, sin = cos[:n], sin[:n]
    if seq_dimension == -3:
        cos, sin = cos[:, None, :], sin[:, None, :]
    return x * cos + rotate_half(x) * sin


class _ApplyRotaryQKV(torch.autograd.Function):
    """In-place rotation of the q and k parts of a packed qkv; the backward rotates the incoming gradient by the
    opposite angle (the transpose of a rotation) and passes the v part through."""

    @staticmethod
    def forward(ctx, qkv, cos_half, sin_half):
        from . import flash_attn_gfx950 as backend
        ctx.save_for_backward(cos_half, sin_half)
        backend.rotary(qkv, qkv, cos_half, sin_half, n_rotated=2)
        ctx.mark_dirty(qkv)
        return qkv

    @staticmethod
    def backward(ctx, grad):
        from . import flash_attn_gfx950 as backend
        cos_half, sin_half = ctx.saved_tensors
        grad = backend.contiguous16(grad)
        return backend.rotary(grad, torch.empty_like(grad), cos_half, sin_half, n_rotated=2, conjugate=True), None, None


def apply_rotary_emb_qkv_(qkv, cos_half, sin_half):
    """Rotates q = qkv[:, :, 0] and k = qkv[:, :, 1] of a packed (batch, seqlen, 3, nheads, headdim) fp16 / bf16 GPU
    tensor IN PLACE by the angles whose cosines / sines are cos_half / sin_half ((>= seqlen, headdim / 2), same dtype):
    the same map as apply_rotary_pos_emb(q, ...), apply_rotary_pos_emb(k, ...) with seq_dimension=-3, products formed in
    fp32 and rounded once.  Differentiable."""
    return _ApplyRotaryQKV.apply(qkv, cos_half, sin_half)


class _QkNormRotary(torch.autograd.Function):
    """q and k normalised, weighted and turned; the backward forms the norms again from q and k, so nothing but the inputs is kept."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos_half, sin_half, positions, seqlen, eps):
        from . import flash_attn_gfx950 as backend
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        backend.qk_norm_rotary(q, k, q_out, k_out, q_weight, k_weight, cos_half, sin_half, positions, seqlen, eps)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos_half, sin_half, positions)
        ctx.seqlen, ctx.eps = seqlen, eps
        return q_out, k_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        from . import flash_attn_gfx950 as backend
        q, k, q_weight, k_weight, cos_half, sin_half, positions = ctx.saved_tensors
        dq_out, dk_out = _kernel_rows(dq_out), _kernel_rows(dk_out)
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        dqw, dkw = backend.qk_norm_rotary_bwd(dq_out, dk_out, q, k, dq, dk, q_weight, k_weight, cos_half, sin_half, positions, ctx.seqlen, ctx.eps)
        return dq, dk, dqw, dkw, None, None, None, None, None


def _kernel_rows(t):
    """t as the kernels read a (rows, heads, headdim) tensor: itself, or a contiguous copy where its strides or its address are not theirs."""
    ok = t.stride(2) == 1 and all(0 <= s < 1 << 24 and s % 8 == 0 for s in t.stride()[:2]) and t.data_ptr() % 16 == 0
    return t if ok else t.clone(memory_format=torch.contiguous_format)  # (contiguous() would hand back one whose address is the fault)


def apply_qk_norm_rotary(q, k, q_weight, k_weight, cos_half=None, sin_half=None, positions=None, eps=1e-6):
    """Queries and keys as attention wants them: every head's vector divided by its root mean square, times the headdim weights, then turned by its
    position (cos_half, sin_half: RotaryEmbedding.half_tables; None: not turned), in one pass, products in fp32, rounded once.
    q: (total, nheads, headdim) or (batch, seqlen, nheads, headdim), k the same with its own number of heads, fp16 or bf16, headdim 16, 32, 64 or 128;
    q_weight, k_weight: (headdim,) in the tensors' dtype or fp32.  positions: int32, one table row for each row of q (entries outside the tables are
    clamped to them); None: the place in the sequence, for tensors with a seqlen dimension or a single packed sequence.
    Returns (q', k'), new tensors; differentiable in q, k and the weights (once)."""
    from . import flash_attn_gfx950 as backend
    done = backend.passes().qk_norm_rotary(q, k, q_weight, k_weight, cos_half, sin_half, positions, eps)
    if done is not None:
        return done
    if q.dim() == 4:
        b, s = q.shape[:2]
        if k.dim() != 4 or tuple(k.shape[:2]) != (b, s):
            raise RuntimeError("q and k must both be (batch, seqlen, heads, headdim)")
        flat = None if positions is None else positions.reshape(-1)
        q2, k2 = _QkNormRotary.apply(_kernel_rows(q.reshape(b * s, *q.shape[2:])), _kernel_rows(k.reshape(b * s, *k.shape[2:])), q_weight, k_weight, cos_half,
                                     sin_half, flat, s, eps)
        return q2.reshape(q.shape), k2.reshape(k.shape)
    if q.dim() != 3 or k.dim() != 3:
        raise RuntimeError("q and k must be (total, heads, headdim) or (batch, seqlen, heads, headdim)")
    return _QkNormRotary.apply(_kernel_rows(q), _kernel_rows(k), q_weight, k_weight, cos_half, sin_half, positions, q.shape[0], eps)


_SHORT = (torch.float16, torch.bfloat16)


def _version(t):
    return 0 if t.is_inference() else t._version


def _inverse_frequencies(dim, device=None):
    return 1.0 / (10000 ** (torch.arange(0, dim, 2, device=device).float() / dim))


class RotaryEmbedding(torch.nn.Module):
    """Rotary embedding of RoFormer (Su et al., arXiv:2104.09864) for queries and keys.  Angles are formed in fp32 at least, also where .half() or .bfloat16()
    have rounded the module's buffer of frequencies."""

    def __init__(self, dim_model: int, *_, **__):
        super().__init__()
        self.register_buffer("inv_freq", _inverse_frequencies(dim_model))
        self._seq_len_cached = None
        self._cos_cached = None
        self._sin_cached = None

    def _apply(self, *args, **kwargs):
        values, wide, was_short = self._values(), self._frequencies(self.inv_freq.device), self.inv_freq.dtype in _SHORT
        out = super()._apply(*args, **kwargs)
        if wide.is_meta or self.inv_freq.is_meta:
            return out
        if self.inv_freq.dtype in _SHORT:
            self._wide_freq, self._wide_of = wide.to(self.inv_freq.device), values
        elif was_short:  # (back from 16 bits)
            self.inv_freq = wide.to(self.inv_freq)
        self._seen = (self.inv_freq, _version(self.inv_freq))  # (moved or cast: the same values)
        return out

    def _values(self):
        """A number for the values of the buffer: another one when it has been loaded or set"""
        seen = self.__dict__.get("_seen")
        if seen is None or seen[0] is not self.inv_freq or seen[1] != _version(self.inv_freq):
            self._seen = (self.inv_freq, _version(self.inv_freq))
            self._count = self.__dict__.get("_count", 0) + 1
        return self._count

    def _frequencies(self, device):
        """The frequencies on `device` in fp32 or more: the buffer's, or, where that has been rounded to 16 bits, what was rounded"""
        freq = self.inv_freq
        if freq.dtype not in _SHORT or freq.is_meta:
            return freq.to(device)
        if self.__dict__.get("_wide_of") != self._values():  # (loaded, or cast past the module: the usual ones rounded, or others)
            wide = _inverse_frequencies(2 * freq.numel(), "cpu").to(freq.device)
            usual = torch.allclose(freq.float(), wide, rtol=torch.finfo(freq.dtype).eps, atol=0.0)
            self._wide_freq, self._wide_of = wide if usual else freq.float(), self._values()
        return self._wide_freq.to(device)

    def _angles(self, positions, device):
        """(positions, dim / 2): an angle for each position 0, 1, .. and each frequency"""
        freq = self._frequencies(device)
        return torch.outer(torch.arange(positions, device=device, dtype=freq.dtype), freq)

    def _update_cos_sin_tables(self, x, seq_dimension=-2):
        seq_len = x.shape[seq_dimension]
        if x.is_cuda and torch.cuda.is_current_stream_capturing():  # (a graph's own: those that are kept go with the next length)
            return self._cos_sin(seq_len, x)
        stale = (seq_len != self._seq_len_cached or self._cos_cached.device != x.device
                 or self._cos_cached.dtype != x.dtype or self.__dict__.get("_cached_values") != self._values())
        if stale:
            self._seq_len_cached, self._cached_values = seq_len, self._values()
            self._cos_cached, self._sin_cached = self._cos_sin(seq_len, x)
        return self._cos_cached, self._sin_cached

    def _cos_sin(self, seq_len, x):
        angles = self._angles(seq_len, x.device)
        return tuple(f(angles).to(x.dtype).repeat_interleave(2, dim=-1) for f in (torch.cos, torch.sin))

    def half_tables(self, qkv):
        """(cos, sin) of shape (seqlen, headdim / 2) for a (batch, seqlen, 3, nheads, headdim) tensor: one entry per rotated
        pair, the form the HIP kernels read.  Same values as forward()'s tables."""
        n, tables, half = qkv.shape[1], self.tables_to(qkv.shape[1], qkv), self.__dict__.get("_half")
        if half is None or half[0] is not tables or half[1] != n:
            self._half = half = (tables, n, (tables[0][:n], tables[1][:n]))  # (in one piece: other threads may ask for other lengths)
        return half[2]

    def tables_to(self, positions, like):
        """(cos, sin) of shape (>= positions, headdim / 2) in `like`'s dtype on its device: tables that grow (to a power of two of rows), for
        positions that grow from call to call.  Those they outgrow are kept, too (all together as many rows again): graphs that read them may be replayed."""
        kept = self.__dict__.setdefault("_tables", {}).setdefault((like.device, like.dtype, self._values()), [])
        have = kept[-1] if kept else None
        if have is None or have[0].shape[0] < positions:
            rows = max(256, 1 << (max(int(positions), 1) - 1).bit_length())
            angles = self._angles(rows, like.device)  # as in _update_cos_sin_tables
            have = (torch.cos(angles).to(like.dtype), torch.sin(angles).to(like.dtype))
            if like.is_cuda and torch.cuda.is_current_stream_capturing():  # (a graph's own: there is nothing in them before it is replayed)
                return have
            if like.is_cuda:  # (the next call may be on another stream; they grow a few times in a process)
                torch.cuda.current_stream(like.device).synchronize()
            kept.append(have)
        return have

    def rotate_qkv_(self, qkv):
        """q and k of a packed (batch, seqlen, 3, nheads, headdim) GPU tensor rotated in place (one HIP kernel); returns
        qkv.  Same tables as forward()."""
        return apply_rotary_emb_qkv_(qkv, *self.half_tables(qkv))

    def forward(self, q: torch.Tensor, k: torch.Tensor, seq_dimension=-2) -> Tuple[torch.Tensor, torch.Tensor]:
        assert seq_dimension in [-2, -3]  # (bs, h, s, d) or (bs, s, h, d)
        cos, sin = self._update_cos_sin_tables(k, seq_dimension=seq_dimension)
        return (apply_rotary_pos_emb(q, cos, sin, seq_dimension), apply_rotary_pos_emb(k, cos, sin, seq_dimension))


class _ApplyRotaryQKV2D(torch.autograd.Function):
    """In-place 2-D rotation of q and k of a packed qkv: channels [0, d/2) by the token's column, [d/2, d) by its row
    (two passes of the same kernel over the two half-channel views, the position of every token given explicitly).  The
    backward applies the opposite rotations to the incoming gradient."""

    @staticmethod
    def _rotate(t, cos_half, sin_half, col_pos, row_pos, conjugate):
        from . import flash_attn_gfx950 as backend
        half = t.shape[-1] // 2
        lo, hi = t[..., :half], t[..., half:]
        backend.rotary(lo, lo, cos_half, sin_half, n_rotated=2, conjugate=conjugate, positions=col_pos)
        backend.rotary(hi, hi, cos_half, sin_half, n_rotated=2, conjugate=conjugate, positions=row_pos)

    @staticmethod
    def forward(ctx, qkv, cos_half, sin_half, col_pos, row_pos):
        ctx.save_for_backward(cos_half, sin_half, col_pos, row_pos)
        _ApplyRotaryQKV2D._rotate(qkv, cos_half, sin_half, col_pos, row_pos, False)
        ctx.mark_dirty(qkv)
        return qkv

    @staticmethod
    def backward(ctx, grad):
        cos_half, sin_half, col_pos, row_pos = ctx.saved_tensors
        grad = grad.clone(memory_format=torch.contiguous_format)
        _ApplyRotaryQKV2D._rotate(grad, cos_half, sin_half, col_pos, row_pos, True)
        return grad, None, None, None, None


class RotaryEmbedding2D(torch.nn.Module):
    """Rotary embedding for a square grid of tokens (seqlen = side * side): the first half of the channels is
    rotated by the column index, the second half by the row index."""

    def __init__(self, dim: int):
        super().__init__()
        assert dim % 4 == 0
        self.rotary_emb1d = RotaryEmbedding(dim // 2)
        self._pos_cached = None

    def rotate_qkv_(self, qkv):
        """q and k of a packed (batch, side * side, 3, nheads, headdim) fp16 / bf16 GPU tensor rotated in place by the HIP
        kernel (headdim a multiple of 16); returns qkv.  Same map as forward() on q and k, products in fp32, one rounding."""
        b, seqlen = qkv.shape[0], qkv.shape[1]
        side = int(math.sqrt(seqlen))
        assert seqlen == side * side
        grid = qkv[:, :side, 0, :, :qkv.shape[-1] // 2]  # (b, side, nheads, headdim / 2): `side` positions per axis
        cos, sin = self.rotary_emb1d._update_cos_sin_tables(grid, seq_dimension=-3)
        return _ApplyRotaryQKV2D.apply(qkv, cos[:, ::2].contiguous(), sin[:, ::2].contiguous(), *self._grid_positions(b, side, qkv))

    def _grid_positions(self, b, side, qkv):
        """(column, row) of every token of b grids"""
        key, have = (b, side, qkv.device), self._pos_cached
        capturing = qkv.is_cuda and torch.cuda.is_current_stream_capturing()
        if capturing or have is None or have[0] != key:
            tok = torch.arange(side * side, device=qkv.device, dtype=torch.int32)
            col = (tok % side).repeat(b).contiguous()
            row = torch.div(tok, side, rounding_mode="floor").to(torch.int32).repeat(b).contiguous()
            have = (key, col, row)
            if not capturing:  # (a graph's own, as in RotaryEmbedding)
                self._pos_cached = have
        return have[1:]

    def forward(self, q: torch.Tensor, k: torch.Tensor, seq_dimension=-2):
        assert seq_dimension in [-2, -3]
        seqlen = q.shape[seq_dimension]
        side = int(math.sqrt(seqlen))
        assert seqlen == side * side
        if seq_dimension == -3:  # (bs, s, h, d) -> (bs, h, s, d)
            q, k = q.transpose(1, 2), k.transpose(1, 2)
        half = q.shape[-1] // 2

        def grid(t):  # (b, nheads, side*side, c) -> (b, nheads, side, side, c)
            return t.reshape(t.shape[0], t.shape[1], side, side, t.shape[-1])

        # first half: position = column (inner grid axis); second half: position = row (outer grid axis)
        q0, k0 = self.rotary_emb1d(grid(q[..., :half]), grid(k[..., :half]), seq_dimension=-2)
        q1, k1 = self.rotary_emb1d(grid(q[..., half:]), grid(k[..., half:]), seq_dimension=-3)
        q_emb = torch.cat([q0.reshape(*q.shape[:-1], half), q1.reshape(*q.shape[:-1], half)], dim=-1)
        k_emb = torch.cat([k0.reshape(*k.shape[:-1], half), k1.reshape(*k.shape[:-1], half)], dim=-1)
        if seq_dimension == -3:
            q_emb, k_emb = q_emb.transpose(1, 2), k_emb.transpose(1, 2)
        return q_emb, k_emb
