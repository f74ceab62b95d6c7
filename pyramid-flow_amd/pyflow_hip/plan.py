"""Per-(unit, stage) sequence plan: token geometry, 3-axis RoPE table and the implicit form of the
reference's block-causal attention mask.  Pure host arithmetic (numpy / torch-CPU), computed once
per (unit, stage) and uploaded; replaces the per-forward `_prepare_pyramid_image_ids`, `EmbedND`
and `[B,1,L,L]` mask construction of modeling_pyramid_flux.py:186-237, 266-270, 318-350.
"""
import numpy as np
import torch
import torch.nn.functional as F


def _axis_pos(n, train_n):
    # modeling_pyramid_flux.py:193-204: linear interpolation of arange(train_n) onto n samples
    if n == train_n:
        return torch.arange(train_n).float()
    return F.interpolate(torch.arange(train_n)[None, None].float(), n, mode="linear")[0, 0]


def image_token_ids(clip_shapes):
    """clip_shapes: list of (t, h, w) LATENT dims, oldest -> newest. Returns ids [L_img,3] float32."""
    th, tw = clip_shapes[-1][1] // 2, clip_shapes[-1][2] // 2
    out, start = [], 0
    for (t, h, w) in clip_shapes:
        h2, w2 = h // 2, w // 2
        ids = torch.zeros(t, h2, w2, 3)
        ids[..., 0] += torch.arange(start, start + t)[:, None, None]
        ids[..., 1] += _axis_pos(h2, th)[None, :, None]
        ids[..., 2] += _axis_pos(w2, tw)[None, None, :]
        out.append(ids.reshape(-1, 3))
        start += t
    return torch.cat(out, 0)


def rope_cos_sin(ids, axes_dim, theta=10000):
    """modeling_pyramid_flux.py:28-57 -> [L, sum(axes)/2, 2] float32 (cos, sin), angles in float64."""
    parts = []
    for i, dim in enumerate(axes_dim):
        scale = torch.arange(0, dim, 2, dtype=torch.float64) / dim
        omega = 1.0 / (theta ** scale)
        ang = ids[:, i].double()[:, None] * omega[None]
        parts.append(torch.stack([torch.cos(ang), torch.sin(ang)], dim=-1))
    return torch.cat(parts, dim=1).float()


class SequencePlan:
    """Geometry of one stage sequence [text(Lt) | clips...] for a CFG batch of B rows."""

    QTILE = 128

    def __init__(self, clip_shapes, enc_mask, axes_dim, device):
        enc_mask = np.asarray(enc_mask.cpu() if isinstance(enc_mask, torch.Tensor) else enc_mask)
        B, Lt = enc_mask.shape
        self.B, self.Lt = B, Lt
        self.clip_shapes = list(clip_shapes)
        self.clip_tokens = [t * (h // 2) * (w // 2) for (t, h, w) in clip_shapes]
        self.L_img = sum(self.clip_tokens)
        self.L = Lt + self.L_img
        self.Lp = (self.L + 63) // 64 * 64
        t, h, w = clip_shapes[-1]
        self.cur = (t, h, w)
        self.n_cur = self.clip_tokens[-1]
        ids = image_token_ids(clip_shapes)
        all_ids = torch.cat([torch.zeros(Lt, 3), ids], 0)
        self.rope = rope_cos_sin(all_ids, axes_dim).contiguous().to(device)
        # ---- implicit mask: valid text must be a prefix (tokenizer pads at the end)
        frame_t = ids[:, 0].numpy().astype(np.int64)
        n_frames = int(frame_t.max()) + 1 if frame_t.size else 0
        counts = np.bincount(frame_t, minlength=n_frames)
        frame_end = Lt + np.cumsum(counts)                       # exclusive end position of frame f
        a_lo = np.zeros((B, self.L), np.int32)
        a_hi = np.zeros((B, self.L), np.int32)
        b_hi = np.zeros((B, self.L), np.int32)
        for b in range(B):
            v = int(enc_mask[b].sum())
            if not (enc_mask[b, :v] == 1).all():
                raise NotImplementedError("encoder_attention_mask must be a prefix of ones (tokenizer right-padding)")
            # valid text rows: valid text + frame(s) with t == 0 ; padded text rows: padded text only
            a_lo[b, :v], a_hi[b, :v], b_hi[b, :v] = 0, v, (frame_end[0] if n_frames else Lt)
            a_lo[b, v:Lt], a_hi[b, v:Lt], b_hi[b, v:Lt] = v, Lt, Lt
            a_lo[b, Lt:], a_hi[b, Lt:] = 0, v
            b_hi[b, Lt:] = frame_end[frame_t]
        nqt = (self.L + self.QTILE - 1) // self.QTILE
        tile_end = np.zeros((B, nqt), np.int32)
        for qt in range(nqt):
            sl = slice(qt * self.QTILE, min((qt + 1) * self.QTILE, self.L))
            tile_end[:, qt] = np.maximum(b_hi[:, sl].max(axis=1), Lt)
        self.a_lo = torch.from_numpy(a_lo).to(device)
        self.a_hi = torch.from_numpy(a_hi).to(device)
        self.b_hi = torch.from_numpy(b_hi).to(device)
        self.tile_kv_end = torch.from_numpy(tile_end).to(device)
        self.host = dict(a_lo=a_lo, a_hi=a_hi, b_hi=b_hi, tile_kv_end=tile_end)

    def dense_mask(self):
        """[B, L, L] bool -- test helper: the mask the intervals stand for."""
        j = np.arange(self.L)[None, None, :]
        a_lo, a_hi, b_hi = (self.host[k][:, :, None] for k in ("a_lo", "a_hi", "b_hi"))
        return np.where(j < self.Lt, (j >= a_lo) & (j < a_hi), j < b_hi)

    def useful_pairs(self, q_row_begin=0):
        """number of unmasked (q, k) pairs summed over the batch for query rows >= q_row_begin (FLOP accounting)."""
        cache = self.__dict__.setdefault("_pairs", {})
        if q_row_begin not in cache:
            h = self.host
            r = q_row_begin
            cache[q_row_begin] = int((h["a_hi"][:, r:] - h["a_lo"][:, r:]).astype(np.int64).sum()
                                     + (h["b_hi"][:, r:] - self.Lt).astype(np.int64).sum())
        return cache[q_row_begin]


class RopeAxes:
    """Rotation of head channels by several position axes, for ops.qk_norm_rope_axes: pair p turns by
    ``pos[axis[p]] * freq[p]`` radians.  ``freq`` float64 and ``axis`` int32, both [n_pairs] device tensors; pairs are channels
    (2 p, 2 p + 1), or (p, p + n_pairs) with ``halves``; channels behind 2 n_pairs pass through.  ``n_axes``: how many axes a position
    has to have at least (None: the axes are on the device and stay unread; one that a position lacks is then taken as its last)."""

    def __init__(self, freq, axis, halves=False, n_axes=None):
        if freq.dtype is not torch.float64 or axis.dtype is not torch.int32 or freq.dim() != 1 or freq.shape != axis.shape:
            raise ValueError("RopeAxes: freq must be float64 [n_pairs] and axis int32 [n_pairs]")
        if not (freq.is_contiguous() and axis.is_contiguous()) or freq.get_device() != axis.get_device():
            raise ValueError("RopeAxes: freq and axis must be contiguous and on one device")
        self.freq, self.axis, self.halves, self.n_pairs, self.n_axes = freq, axis, bool(halves), freq.numel(), n_axes

    @classmethod
    def build(cls, axes_dim, device, theta=10000.0, halves=False):
        """``axes_dim`` channels per axis, each axis with its own spectrum theta^(-2 k / dim) (as rope_cos_sin)."""
        if any(d <= 0 or d % 2 for d in axes_dim):
            raise ValueError("RopeAxes: channels per axis must be positive and even")
        freq = torch.cat([1.0 / (theta ** (torch.arange(0, d, 2, dtype=torch.float64) / d)) for d in axes_dim])
        axis = torch.cat([torch.full((d // 2,), n, dtype=torch.int32) for n, d in enumerate(axes_dim)])
        return cls(freq.to(device), axis.to(device), halves, n_axes=len(axes_dim))


class KeyRanges:
    """The keys each row sees, for ops.attention_ranges: [a_lo, a_hi) and, if given, [b_lo, b_hi) -- int32 [B][Lq] (or [1][Lq]:
    shared by the batch) device tensors.  A row with two empty ranges sees nothing."""

    def __init__(self, a_lo, a_hi, b_lo=None, b_hi=None):
        if (b_lo is None) != (b_hi is None):
            raise ValueError("KeyRanges: a second range needs its start and its end")
        shape, device = a_lo.shape, a_lo.get_device()
        for t in (a_lo, a_hi) if b_lo is None else (a_lo, a_hi, b_lo, b_hi):
            if t.dtype is not torch.int32 or t.shape != shape or len(shape) != 2 or t.get_device() != device or not t.is_contiguous():
                raise ValueError("KeyRanges: ranges must be contiguous int32 [B or 1][Lq] tensors of one shape on one device")
        self.a_lo, self.a_hi, self.b_lo, self.b_hi = a_lo, a_hi, b_lo, b_hi

    @classmethod
    def _of(cls, device, *arrays):
        return cls(*[None if a is None else torch.from_numpy(np.ascontiguousarray(np.atleast_2d(a), dtype=np.int32)).to(device)
                     for a in arrays])

    @classmethod
    def causal(cls, Lq, Lk, device):
        """row i is key Lk - Lq + i and sees the keys up to itself"""
        return cls._of(device, np.zeros(Lq), np.arange(Lq) + (Lk - Lq) + 1)

    @classmethod
    def padded(cls, lengths, Lq, device):
        """every row of batch entry b sees the first lengths[b] keys"""
        hi = np.repeat(np.asarray(lengths)[:, None], Lq, 1)
        return cls._of(device, np.zeros_like(hi), hi)

    @classmethod
    def documents(cls, lengths, L, device, causal=False):
        """documents packed one behind the other into L rows; rows behind the last one see nothing"""
        lengths = np.asarray(lengths, dtype=np.int64)
        if (lengths < 0).any() or lengths.sum() > L:
            raise ValueError("KeyRanges.documents: lengths must be >= 0 and fit into L")
        end = np.cumsum(lengths)
        lo, hi = np.zeros(L, np.int64), np.zeros(L, np.int64)
        used = int(lengths.sum())
        lo[:used], hi[:used] = np.repeat(end - lengths, lengths), np.repeat(end, lengths)
        if causal:
            hi[:used] = np.arange(used) + 1
        return cls._of(device, lo, hi)

    @classmethod
    def prefix(cls, prefix, L, device):
        """the first prefix[b] keys are seen by all rows, later ones by the rows from themselves on"""
        return cls._of(device, np.zeros((len(prefix), L)), np.maximum(np.arange(L)[None] + 1, np.minimum(np.asarray(prefix), L)[:, None]))

    @classmethod
    def from_key_mask(cls, mask, Lq, device):
        """mask [B][Lk], nonzero = visible to every row: at most two runs of visible keys per batch entry"""
        mask = np.asarray(mask.cpu() if isinstance(mask, torch.Tensor) else mask) != 0
        out = np.zeros((4, mask.shape[0], Lq), np.int64)
        for b, row in enumerate(mask):
            edges = np.flatnonzero(np.diff(np.concatenate([[0], row.astype(np.int8), [0]])))
            if len(edges) > 4:
                raise NotImplementedError("KeyRanges.from_key_mask: more than two runs of visible keys")
            for n, e in enumerate(edges):
                out[n, b] = e
        return cls._of(device, *out)

    @classmethod
    def from_plan(cls, plan):
        """the joint text-video mask of a SequencePlan"""
        return cls(plan.a_lo, plan.a_hi, torch.full_like(plan.b_hi, plan.Lt), plan.b_hi)

    def pairs(self, B, Lk):
        """visible (row, key) pairs of a head, all B batch entries together, over Lk keys (read back from the device)"""
        lo, hi = (t.long().clamp(0, Lk) for t in (self.a_lo, self.a_hi))
        n = (hi - lo).clamp(min=0)
        if self.b_lo is not None:
            lo2, hi2 = (t.long().clamp(0, Lk) for t in (self.b_lo, self.b_hi))
            n2 = (hi2 - lo2).clamp(min=0)
            n = n + n2 - (torch.minimum(hi, hi2) - torch.maximum(lo, lo2)).clamp(min=0) * (n > 0) * (n2 > 0)
        return int(n.sum()) * (B if n.shape[0] == 1 else 1)

    def dense_mask(self, Lk):
        """[B or 1, Lq, Lk] bool -- test helper: the mask the ranges stand for"""
        j = torch.arange(Lk, device=self.a_lo.device)
        seen = (j >= self.a_lo[..., None]) & (j < self.a_hi[..., None])
        if self.b_lo is not None:
            seen |= (j >= self.b_lo[..., None]) & (j < self.b_hi[..., None])
        return seen
