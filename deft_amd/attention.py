"""Attention-layer operators over tokens: detections (or map cells) at positions (frame, y, x).

The second kind of sequence model next to engine.LstmPlan: where that one carries a track's history in an LSTM state row (kalman_filter_lstm.py:9-29),
an attention layer reads the history itself.  Three operators, each one call of the C ABI (include/deft_hip.h DeftRotary, DeftAttn):

  AttentionPlan.rotate        rotary positions with several axes on queries and keys
  AttentionPlan.norm_rotate   RMS norm of every query / key head and the rotation in one pass; keys and values into cache rows
  AttentionPlan.attend        causal attention, grouped heads, packed sequences of different lengths or single tokens over a cache

Tensors are fp32, fp16 or bf16, [tokens][heads][head_dim] with any token and head stride that is a multiple of 16 bytes (views of one projection
buffer need no copy).  Every call is asynchronous on the current stream of the plan's device; outputs and workspaces are allocated per call by torch's
stream-ordered allocator, so calls on several streams and captured graphs share nothing.  Forward only, like the rest of the package; refusals raise
DeftHipError.
"""
import ctypes as C
import math

import torch

from . import hiplib
from .engine import _Plan
from .hiplib import AttnDesc, DeftHipError, RotaryDesc

_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _refuse(cond, *msg):
    if cond:
        raise DeftHipError("attention: " + msg[0] % msg[1:])


class AttentionPlan(_Plan):
    """heads / kv_heads / head_dim of the layer (kv_heads divides heads; head h reads kv head h // (heads // kv_heads)).

    axes: number of rotated pairs of each position axis, e.g. (8, 12, 12) for (frame, y, x) and head_dim 64; pairs of an axis are neighbours and pair
    i turns by pos[axis] * freq[i].  freq (float64, one per pair) defaults to theta ** (-i / pairs) over all pairs; axis_of_pair overrides which
    axis a pair takes.  A pair is elements (i, i + pairs), or (2i, 2i + 1) with adjacent=True; elements behind the 2 * pairs first are not turned.
    q_weight / k_weight [head_dim]: weights of the norms (None = 1).  scale: of the scores, 1 / sqrt(head_dim) by default."""

    def __init__(self, heads, kv_heads, head_dim, axes=None, theta=10000.0, freq=None, axis_of_pair=None, adjacent=False, q_weight=None, k_weight=None,
                 eps=1e-6, scale=None, device="cuda", lib=None):
        super().__init__(device, lib)
        _refuse(heads < 1 or kv_heads < 1 or heads % kv_heads, "heads=%d is not a multiple of kv_heads=%d", heads, kv_heads)
        self.heads, self.kv_heads, self.head_dim = int(heads), int(kv_heads), int(head_dim)
        self.scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
        self.eps, self.adjacent = float(eps), bool(adjacent)
        self.device = torch.empty(0, device=self.device).device          # with its index: tensors and launches belong to THIS device
        self.pairs = 0
        if axes is not None:
            axes = [int(n) for n in axes]
            _refuse(not axes or min(axes) < 0 or sum(axes) < 1 or 2 * sum(axes) > head_dim, "axes=%s: 1 .. %d pairs in all", axes, head_dim // 2)
            self.pairs, self.naxes = sum(axes), len(axes)
            axis = [a for a, n in enumerate(axes) for _ in range(n)] if axis_of_pair is None else [int(a) for a in axis_of_pair]
            _refuse(len(axis) != self.pairs or min(axis) < 0 or max(axis) >= self.naxes, "axis_of_pair: %d values in 0 .. %d", self.pairs, self.naxes - 1)
            f = torch.tensor([theta ** (-i / self.pairs) for i in range(self.pairs)], dtype=torch.float64) if freq is None else \
                torch.as_tensor(freq).detach().to(dtype=torch.float64, device="cpu")
            _refuse(tuple(f.shape) != (self.pairs,), "freq: one value for each of the %d pairs", self.pairs)
            self.freq = self.dev(f)
            self.axis = self.dev(torch.tensor(axis, dtype=torch.int32))
        self.q_weight, self.k_weight = self._weight("q_weight", q_weight), self._weight("k_weight", k_weight)

    def _weight(self, name, w):
        if w is None:
            return None
        _refuse(tuple(w.shape) != (self.head_dim,), "%s has shape %s, wanted [%d]", name, tuple(w.shape), self.head_dim)
        return self.dev(w.detach().to(torch.float32).clone())

    def _rows(self, name, x, heads, dtype, tokens=None, ndim=3):
        """Refuses what is not [tokens][heads][head_dim] (ndim 4: [slots][rows][heads][head_dim]) rows of `dtype` on the plan's device."""
        _refuse(not isinstance(x, torch.Tensor), "%s is not a tensor", name)
        shape = x.shape
        _refuse(len(shape) != ndim or shape[-2] != heads or shape[-1] != self.head_dim, "%s has shape %s, wanted %s[%d][%d]", name, tuple(shape),
                "[tokens]" if ndim == 3 else "[slots][rows]", heads, self.head_dim)
        _refuse(x.dtype is not dtype, "%s is %s, wanted %s", name, x.dtype, dtype)
        _refuse(x.device != self.device, "%s is on %s, the plan on %s", name, x.device, self.device)
        _refuse(tokens is not None and shape[0] != tokens, "%s has %d tokens, wanted %d", name, shape[0], tokens)
        st = x.stride()
        _refuse(st[-1] != 1 and shape[-1] > 1, "%s: elements of a head must be contiguous", name)
        return [0 if n == 1 else s for n, s in zip(shape, st)]           # (the stride of a one-long dimension says nothing)

    def _ints(self, name, x, n, dtype=torch.int32):
        _refuse(not isinstance(x, torch.Tensor) or x.dtype is not dtype or x.dim() != 1 or x.shape[0] != n or x.device != self.device or not x.is_contiguous(),
                "%s: a contiguous %s tensor of %d values on %s", name, dtype, n, self.device)
        return x.data_ptr()

    def _launch(self, entry, desc):
        if self.device.type == "cuda" and torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                self.lib.call(entry, C.byref(desc), self._stream())
        else:
            self.lib.call(entry, C.byref(desc), self._stream())

    # ---- rotary positions, norms ---------------------------------------------------------------------------------------------------------
    def rotate(self, q, k, pos, v=None, cache=None, row=None, out=None, inverse=False):
        """Turns q [T][heads][D] and k [T][kv_heads][D] (None: queries only) by their positions pos [T][axes] (int32, or float32 for sub-pixel
        centres).  Returns (q', k'): new tensors, or `out` = (q_out, k_out) (which may be q and k themselves).  cache = (k_cache, v_cache) with
        row [T] int32: token t's key -- and value, with v [T][kv_heads][D] -- are written to row row[t] of the caches ([rows] or [slots][rows]
        [kv_heads][D]; a row outside is skipped, no two tokens may share one) and k' is the key cache.  inverse: turns back."""
        return self._rotary(q, k, pos, v, cache, row, out, inverse, False)

    def norm_rotate(self, q, k, pos, v=None, cache=None, row=None, out=None):
        """rotate() of the RMS-normed heads: x * weight / sqrt(mean(x^2) + eps) per head, then the rotation, one pass, one rounding."""
        return self._rotary(q, k, pos, v, cache, row, out, False, True)

    def _rotary(self, q, k, pos, v, cache, row, out, inverse, norm):
        _refuse(not self.pairs, "the plan was made without axes")
        H, Hk, D, dt = self.heads, self.kv_heads, self.head_dim, getattr(q, "dtype", None)
        _refuse(dt not in _DTYPE, "q is %s, wanted float32, float16 or bfloat16", dt)
        sq = self._rows("q", q, H, dt)
        T = q.shape[0]
        _refuse(not isinstance(pos, torch.Tensor) or pos.dtype not in (torch.int32, torch.float32) or pos.device != self.device
                or tuple(pos.shape) != (T, self.naxes) or not pos.is_contiguous(),
                "pos: a contiguous int32 or float32 tensor [%d][%d] on %s", T, self.naxes, self.device)
        _refuse(k is None and (v is not None or cache is not None), "v and cache need k")
        _refuse((cache is None) != (row is None), "cache and row come together")
        _refuse(cache is None and v is not None, "v needs a cache")
        d = RotaryDesc()
        q_out, k_out = out if out is not None else (None, None)
        if q_out is None:
            q_out = torch.empty((T, H, D), dtype=dt, device=self.device)
        so = self._rows("q_out", q_out, H, dt, T)
        d.q, d.q_out, d.pos, d.freq, d.axis = q.data_ptr(), q_out.data_ptr(), pos.data_ptr(), self.freq.data_ptr(), self.axis.data_ptr()
        d.ldq, d.hsq, d.ldqo, d.hsqo = sq[0], sq[1], so[0], so[1]
        if k is not None:
            sk = self._rows("k", k, Hk, dt, T)
            d.k, d.ldk, d.hsk = k.data_ptr(), sk[0], sk[1]
            if cache is not None:
                _refuse(k_out is not None, "out[1] and a cache are one too many")
                k_out, v_cache = cache
                rows, d.k_out, d.ldko, d.hsko = self._cache_rows("k_cache", k_out, dt)
                _refuse((v is None) != (v_cache is None), "v and v_cache come together")
                if v is not None:
                    sv = self._rows("v", v, Hk, dt, T)
                    d.v, d.ldv, d.hsv = v.data_ptr(), sv[0], sv[1]
                    vrows, d.v_out, d.ldvo, d.hsvo = self._cache_rows("v_cache", v_cache, dt)
                    _refuse(vrows != rows, "k_cache has %d rows, v_cache %d", rows, vrows)
                d.row, d.rows = self._ints("row", row, T), rows
            else:
                if k_out is None:
                    k_out = torch.empty((T, Hk, D), dtype=dt, device=self.device)
                sk = self._rows("k_out", k_out, Hk, dt, T)
                d.k_out, d.ldko, d.hsko = k_out.data_ptr(), sk[0], sk[1]
        d.T, d.Hq, d.Hk, d.D, d.R, d.A = T, H, Hk, D, self.pairs, self.naxes
        d.dtype, d.pos_float, d.adjacent, d.inverse, d.norm, d.eps = _DTYPE[dt], pos.dtype is torch.float32, self.adjacent, inverse, norm, self.eps
        if norm:
            d.q_weight = self.q_weight.data_ptr() if self.q_weight is not None else None
            d.k_weight = self.k_weight.data_ptr() if self.k_weight is not None else None
        if T:
            self._launch("deft_rotary", d)
        return q_out, k_out

    def _cache_rows(self, name, x, dt):
        """(rows, address, row stride, head stride) of a cache [rows][kv_heads][D] or [slots][rows][kv_heads][D] whose slots follow each other."""
        nd = x.dim() if isinstance(x, torch.Tensor) else 0
        st = self._rows(name, x, self.kv_heads, dt, ndim=4 if nd == 4 else 3)
        if nd == 4:
            S, cap = x.shape[0], x.shape[1]
            _refuse(S > 1 and cap > 1 and st[0] != cap * st[1], "%s: the rows of its slots must follow each other", name)
            rows, ld = S * cap, st[1] if cap > 1 else st[0]
        else:
            rows, ld = x.shape[0], st[0]
        _refuse(rows < 1, "%s is empty", name)
        return rows, x.data_ptr(), ld, st[-2]

    # ---- attention -----------------------------------------------------------------------------------------------------------------------
    def attend(self, q, k, v, q_start, k_start=None, slot=None, k_len=None, causal=True, max_k=None, lse=False, out=None):
        """softmax(scale * q k^T) v of B sequences of different lengths; returns o [Tq][heads][D] (or `out`; it must not overlap k or v).

        q [Tq][heads][D]; q_start [B + 1] int32 on the device: sequence b owns the query rows q_start[b] .. q_start[b + 1] - 1 (n of them).
        k, v [Tk][kv_heads][D]: packed; sequence b's keys are the k_len[b] rows from k_start[b] on (both default to the queries' own rows).
        k, v [slots][cap][kv_heads][D]: a cache; its keys are the k_len[b] first rows of slot slot[b].
        causal: query i of n sees the keys j <= m - n + i of its m (a lone new token sees all of them).  Rows that see no key give 0; rows of no
        sequence are not written.  Starts, lengths and slots are int32 device tensors, clamped to the tensors by the kernel; max_k (host): an
        estimate of the longest m (default: the cap or the number of key rows), which steers only how the work is split.
        lse=True: returns (o, lse [Tq][heads] float32), the log of each row's sum of exponentials (-inf where it sees no key)."""
        H, Hk, D, dt = self.heads, self.kv_heads, self.head_dim, getattr(q, "dtype", None)
        _refuse(dt not in _DTYPE, "q is %s, wanted float32, float16 or bfloat16", dt)
        sq = self._rows("q", q, H, dt)
        Tq = q.shape[0]
        _refuse(not isinstance(q_start, torch.Tensor) or q_start.dim() != 1 or q_start.shape[0] < 1, "q_start: B + 1 values")
        B = q_start.shape[0] - 1
        paged = isinstance(k, torch.Tensor) and k.dim() == 4
        sk = self._rows("k", k, Hk, dt, ndim=4 if paged else 3)
        sv = self._rows("v", v, Hk, dt, ndim=4 if paged else 3)
        _refuse(k.shape != v.shape, "k has shape %s, v %s", tuple(k.shape), tuple(v.shape))
        d = AttnDesc()
        d.q_start = self._ints("q_start", q_start, B + 1)
        if paged:
            _refuse(slot is None or k_len is None or k_start is not None, "a cache [slots][cap] needs slot and k_len, and no k_start")
            d.k_start, d.ssk, d.ssv, d.cap = self._ints("slot", slot, B), sk[0], sv[0], k.shape[1]
            longest = k.shape[1]
        else:
            _refuse(slot is not None, "slot needs a cache [slots][cap][kv_heads][head_dim]")
            if k_start is not None:
                d.k_start = self._ints("k_start", k_start, B)
            longest = k.shape[0]
        if k_len is not None:
            d.k_len = self._ints("k_len", k_len, B)
        if out is None:
            out = torch.empty((Tq, H, D), dtype=dt, device=self.device)
        so = self._rows("out", out, H, dt, Tq)
        logs = torch.empty((Tq, H), dtype=torch.float32, device=self.device) if lse else None
        if Tq and B:
            empty = not k.numel()                               # nothing to read: every row of a sequence becomes 0
            d.slots, d.cap = (0, 0) if empty else (k.shape[0], d.cap)
            if empty:
                d.k_start = d.k_len = None
            d.q, d.k, d.v, d.o = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
            d.lse = logs.data_ptr() if lse else None
            d.ldq, d.hsq, d.ldk, d.hsk = sq[0], sq[1], sk[-3], sk[-2]
            d.ldv, d.hsv, d.ldo, d.hso = sv[-3], sv[-2], so[0], so[1]
            d.Tq, d.B, d.Hq, d.Hk, d.D, d.dtype, d.causal, d.scale = Tq, B, H, Hk, D, _DTYPE[dt], bool(causal), self.scale
            d.max_k = longest if max_k is None else max(0, min(int(max_k), 0x7fffffff))
            n = self.lib.value("deft_attn_ws_floats", C.byref(d))
            if n > 0:
                ws = torch.empty(n, dtype=torch.float32, device=self.device)       # (stream-ordered: free for the next call once this one is queued)
                d.ws, d.ws_floats = ws.data_ptr(), n
            self._launch("deft_attn", d)
        return (out, logs) if lse else out
