"""Attention-layer operators over tokens: detections (or map cells) at positions (frame, y, x).

Operators for a caller's own attention model, where engine.LstmPlan carries a track's history in an LSTM state row (kalman_filter_lstm.py:9-29) and an
attention layer reads the history itself.  Three operators, each one call of the C ABI (include/deft_hip.h DeftRotary, DeftAttn):

  AttentionPlan.rotate        rotary positions with several axes on queries and keys
  AttentionPlan.norm_rotate   RMS norm of every query / key head and the rotation in one pass; keys and values into cache rows
  AttentionPlan.attend        causal attention, grouped heads, packed sequences of different lengths or single tokens over a cache

Tensors are fp32, fp16 or bf16, [tokens][heads][head_dim] with any token and head stride that is a multiple of 16 bytes (views of one projection
buffer need no copy).  Every call is asynchronous on the current stream of the plan's device; outputs and workspaces are allocated per call by torch's
stream-ordered allocator, so calls on several streams and captured graphs share nothing.  Forward only, like the rest of the package; refusals raise
DeftHipError.
"""
import math
import struct

import torch
from torch.autograd import forward_ad

from .engine import _Plan
from .hiplib import DeftHipError, _raw_stream

_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_current_device = torch.cuda.current_device
# DeftRotary and DeftAttn packed in one call each (field order and layout of hiplib.RotaryDesc / AttnDesc): a call's host time is what counts where a
# launch is a few microseconds, and setting forty ctypes fields one by one costs as much as such a launch
_ROTARY = struct.Struct("@12P13q11if0q")
_ATTN = struct.Struct("@9P11q10if0q")
_SPLIT_KEYS = 256          # no kernel splits the keys of a row below this many (csrc/attn.hip choose()): no workspace to ask for


def _refuse(cond, *msg):
    if cond:
        raise DeftHipError("attention: " + msg[0] % msg[1:])


def _no_gradient(name, x):
    """Refuses x that needs a gradient (under torch.no_grad it needs none) or carries a forward-mode tangent: neither would come out again."""
    if isinstance(x, torch.Tensor):
        _refuse(x.requires_grad and torch.is_grad_enabled(), "%s requires a gradient: these operators are forward only (torch.no_grad, or detach)", name)
        _refuse(forward_ad._current_level >= 0 and x.is_floating_point() and forward_ad.unpack_dual(x).tangent is not None,
                "%s carries a tangent: these operators are forward only", name)


class AttentionPlan(_Plan):
    """heads / kv_heads / head_dim of the layer (kv_heads divides heads; head h reads kv head h // (heads // kv_heads)).

    axes: number of rotated pairs of each position axis, e.g. (8, 12, 12) for (frame, y, x) and head_dim 64; pairs of an axis are neighbours and pair
    i turns by pos[axis] * freq[i].  freq (float64, one per pair) defaults to theta ** (-i / pairs) over all pairs; axis_of_pair overrides which
    axis a pair takes.  A pair is elements (i, i + pairs), or (2i, 2i + 1) with adjacent=True; elements behind the 2 * pairs first are not turned.
    q_weight / k_weight [head_dim]: weights of the norms (None = 1).  scale: of the scores, 1 / sqrt(head_dim) by default.
    `attend` takes head_dim 32, 64, 96 or 128; the rotations multiples of 16 (fp32: 8) up to 256, with pairs in multiples of 8 (fp32: 4).
    The plan keeps copies of freq and the weights as they are when it is made."""

    def __init__(self, heads, kv_heads, head_dim, axes=None, theta=10000.0, freq=None, axis_of_pair=None, adjacent=False, q_weight=None, k_weight=None,
                 eps=1e-6, scale=None, device="cuda", lib=None):
        super().__init__(device, lib)
        # what no call could take (types and single operators ask for more: include/deft_hip.h)
        _refuse(heads < 1 or kv_heads < 1 or heads % kv_heads or heads > 4096, "heads=%d is not a multiple of kv_heads=%d, or above 4096", heads, kv_heads)
        _refuse(head_dim < 8 or head_dim > 256 or head_dim % 8, "head_dim D=%d (a multiple of 8, at most 256)", head_dim)
        _refuse(scale is not None and not 2.0 ** -126 <= scale <= 2.0 ** 126, "scale=%g (2^-126 .. 2^126)", scale)
        _refuse(not 0.0 <= eps < math.inf, "eps=%g", eps)
        self.heads, self.kv_heads, self.head_dim = int(heads), int(kv_heads), int(head_dim)
        self.scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
        self.eps, self.adjacent = float(eps), bool(adjacent)
        at = torch.empty(0, device=self.device)                          # (with its index: tensors and launches belong to THIS device)
        self.device, self._index = at.device, at.get_device()            # -1: host memory, the unit-test build
        self.pairs = 0
        if axes is not None:
            axes = [int(n) for n in axes]
            _refuse(not axes or min(axes) < 0 or sum(axes) < 1 or 2 * sum(axes) > head_dim, "axes=%s: 1 .. %d pairs in all", axes, head_dim // 2)
            self.pairs, self.naxes = sum(axes), len(axes)
            _refuse(self.naxes > 8, "%d axes (at most 8)", self.naxes)
            _refuse(self.pairs % 4, "R=%d pairs (a multiple of 4, of 8 for 16-bit types)", self.pairs)
            axis = [a for a, n in enumerate(axes) for _ in range(n)] if axis_of_pair is None else [int(a) for a in axis_of_pair]
            _refuse(len(axis) != self.pairs or min(axis) < 0 or max(axis) >= self.naxes, "axis_of_pair: %d values in 0 .. %d", self.pairs, self.naxes - 1)
            _no_gradient("freq", freq)
            f = torch.tensor([theta ** (-i / self.pairs) for i in range(self.pairs)], dtype=torch.float64) if freq is None else \
                torch.as_tensor(freq).detach().to(dtype=torch.float64, device="cpu")
            _refuse(tuple(f.shape) != (self.pairs,), "freq: one value for each of the %d pairs", self.pairs)
            self.freq = self.dev(f)
            self.axis = self.dev(torch.tensor(axis, dtype=torch.int32))
            self._freq_ptr, self._axis_ptr = self.freq.data_ptr(), self.axis.data_ptr()
        self.q_weight, self.k_weight = self._weight("q_weight", q_weight), self._weight("k_weight", k_weight)
        self._qw_ptr = 0 if self.q_weight is None else self.q_weight.data_ptr()
        self._kw_ptr = 0 if self.k_weight is None else self.k_weight.data_ptr()
        if any(w is not None and w.is_cuda for w in (q_weight, k_weight)):
            torch.cuda.current_stream(self.device).synchronize()         # (copies from host memory have arrived; calls may come on any stream)

    def _weight(self, name, w):
        if w is None:
            return None
        _no_gradient(name, w)
        _refuse(tuple(w.shape) != (self.head_dim,), "%s has shape %s, wanted [%d]", name, tuple(w.shape), self.head_dim)
        return self.dev(w.detach().to(torch.float32).clone())

    def _rows(self, name, x, heads, dtype, tokens=None):
        """(token stride, head stride) of x [tokens][heads][head_dim]; refuses what is not such rows of `dtype` on the plan's device."""
        try:
            T, h, D = x.shape
            ld, hs, one = x.stride()
            if h == heads and D == self.head_dim and x.dtype is dtype and one == 1 and (tokens is None or T == tokens) and x.get_device() == self._index \
                    and not x.requires_grad:
                return D if T == 1 else ld, D if h == 1 else hs          # (the stride of a one-long dimension says nothing)
        except (AttributeError, ValueError, TypeError):
            pass
        return self._not_rows(name, x, heads, dtype, tokens, "[tokens]")

    def _slots(self, name, x, dtype):
        """(slot stride, row stride, head stride) of a cache x [slots][rows][kv_heads][head_dim]."""
        try:
            S, cap, h, D = x.shape
            ss, ld, hs, one = x.stride()
            if h == self.kv_heads and D == self.head_dim and x.dtype is dtype and one == 1 and x.get_device() == self._index and not x.requires_grad:
                return 0 if S == 1 else ss, D if cap == 1 else ld, D if h == 1 else hs
        except (AttributeError, ValueError, TypeError):
            pass
        return self._not_rows(name, x, self.kv_heads, dtype, None, "[slots][rows]")

    def _not_rows(self, name, x, heads, dtype, tokens, lead):
        _refuse(not isinstance(x, torch.Tensor), "%s is not a tensor", name)
        _refuse(x.dim() != (3 if lead == "[tokens]" else 4) or x.shape[-2] != heads or x.shape[-1] != self.head_dim, "%s has shape %s, wanted %s[%d][%d]", name,
                tuple(x.shape), lead, heads, self.head_dim)
        _refuse(x.dtype is not dtype, "%s is %s, wanted %s", name, x.dtype, dtype)
        _refuse(x.get_device() != self._index, "%s is on %s, the plan on %s", name, x.device, self.device)
        _refuse(tokens is not None and x.shape[0] != tokens, "%s has %d tokens, wanted %s", name, x.shape[0], tokens)
        _refuse(x.stride(-1) != 1, "%s: elements of a head must be contiguous", name)
        _no_gradient(name, x)
        return self._rows(name, x.detach(), heads, dtype, tokens) if lead == "[tokens]" else self._slots(name, x.detach(), dtype)

    def _ints(self, name, x, n):
        """Address of n int32 values on the plan's device."""
        if not (isinstance(x, torch.Tensor) and x.dtype is torch.int32 and x.dim() == 1 and x.shape[0] == n and x.get_device() == self._index
                and x.is_contiguous()):
            _refuse(True, "%s: a contiguous int32 tensor of %d values on %s", name, n, self.device)
        return x.data_ptr()

    def _launch(self, entry, desc):
        if self._index < 0:
            self.lib.call(entry, desc, None)
        elif _current_device() == self._index:
            self.lib.call(entry, desc, _raw_stream(self._index) if _raw_stream is not None else self._stream().value)
        else:
            with torch.cuda.device(self._index):
                self.lib.call(entry, desc, self._stream().value)

    # ---- rotary positions, norms ---------------------------------------------------------------------------------------------------------
    def rotate(self, q, k, pos, v=None, cache=None, row=None, out=None, inverse=False):
        """Turns q [T][heads][D] and k [T][kv_heads][D] (None: queries only) by their positions pos [T][axes] (int32, or float32 for sub-pixel
        centres).  Returns (q', k'): new tensors, or `out` = (q_out, k_out) (which may be q and k themselves, and must not overlap them otherwise).  cache = (k_cache, v_cache) with
        row [T] int32: token t's key -- and value, with v [T][kv_heads][D] -- are written to row row[t] of the caches ([rows] or [slots][rows]
        [kv_heads][D]; a row outside is skipped, no two tokens may share one, the caches overlap no input) and k' is the key cache.  inverse: turns back."""
        return self._rotary(q, k, pos, v, cache, row, out, inverse, False)

    def norm_rotate(self, q, k, pos, v=None, cache=None, row=None, out=None):
        """rotate() of the RMS-normed heads: x * weight / sqrt(mean(x^2) + eps) per head, then the rotation, one pass, one rounding."""
        return self._rotary(q, k, pos, v, cache, row, out, False, True)

    def _rotary(self, q, k, pos, v, cache, row, out, inverse, norm):
        _refuse(not self.pairs, "the plan was made without axes")
        H, Hk, D, dt = self.heads, self.kv_heads, self.head_dim, getattr(q, "dtype", None)
        if dt not in _DTYPE:
            _refuse(True, "q is %s, wanted float32, float16 or bfloat16", dt)
        ldq, hsq = self._rows("q", q, H, dt)
        T = q.shape[0]
        if T > 1 << 30:
            _refuse(True, "q has %d tokens (at most 2^30)", T)
        if forward_ad._current_level >= 0:
            for name, x in (("q", q), ("k", k), ("v", v), ("pos", pos), *zip(("k_cache", "v_cache"), cache or ()), *zip(("q_out", "k_out"), out or ())):
                _no_gradient(name, x)
        pt = getattr(pos, "dtype", None)
        if not ((pt is torch.int32 or pt is torch.float32) and pos.shape == (T, self.naxes) and pos.get_device() == self._index and pos.is_contiguous()):
            _refuse(True, "pos: a contiguous int32 or float32 tensor [%d][%d] on %s", T, self.naxes, self.device)
        if pos.requires_grad:
            _no_gradient("pos", pos)
        q_out, k_out = out if out is not None else (None, None)
        if q_out is None:
            q_out, ldqo, hsqo = q.new_empty((T, H, D)), H * D, D
        else:
            ldqo, hsqo = self._rows("q_out", q_out, H, dt, T)
        kp = vp = kop = vop = rowp = ldk = hsk = ldv = hsv = ldko = hsko = ldvo = hsvo = rows = 0
        if k is None:
            _refuse(v is not None or cache is not None or k_out is not None, "v, a cache and out[1] need k")
        else:
            ldk, hsk = self._rows("k", k, Hk, dt, T)
            kp = k.data_ptr()
            if cache is None:
                _refuse(row is not None, "cache and row come together")
                _refuse(v is not None, "v needs a cache")
                if k_out is None:
                    k_out, ldko, hsko = k.new_empty((T, Hk, D)), Hk * D, D
                else:
                    ldko, hsko = self._rows("k_out", k_out, Hk, dt, T)
            else:
                _refuse(row is None, "cache and row come together")
                _refuse(k_out is not None, "out[1] and a cache are one too many")
                k_out, v_cache = cache
                rows, ldko, hsko = self._cache_rows("k_cache", k_out, dt)
                if (v is None) != (v_cache is None):
                    _refuse(True, "v and v_cache come together")
                if v is not None:
                    ldv, hsv = self._rows("v", v, Hk, dt, T)
                    vrows, ldvo, hsvo = self._cache_rows("v_cache", v_cache, dt)
                    if vrows != rows:
                        _refuse(True, "k_cache has %d rows, v_cache %d", rows, vrows)
                    vp, vop = v.data_ptr(), v_cache.data_ptr()
                rowp = self._ints("row", row, T)
            kop = k_out.data_ptr()
        if T:
            self._launch("deft_rotary", _ROTARY.pack(
                q.data_ptr(), kp, vp, q_out.data_ptr(), kop, vop, pos.data_ptr(), self._freq_ptr, self._axis_ptr, self._qw_ptr if norm else 0,
                self._kw_ptr if norm else 0, rowp, ldq, hsq, ldk, hsk, ldv, hsv, ldqo, hsqo, ldko, hsko, ldvo, hsvo, rows,
                T, H, Hk, D, self.pairs, self.naxes, _DTYPE[dt], pt is torch.float32, self.adjacent, inverse, norm, self.eps))
        return q_out, k_out

    def _cache_rows(self, name, x, dt):
        """(rows, row stride, head stride) of a cache [rows][kv_heads][D] or [slots][rows][kv_heads][D] whose slots follow each other."""
        if isinstance(x, torch.Tensor) and x.dim() == 4:
            ss, ld, hs = self._slots(name, x, dt)
            S, cap = x.shape[0], x.shape[1]
            if S > 1 and cap > 1 and ss != cap * ld:
                _refuse(True, "%s: the rows of its slots must follow each other", name)
            rows, ld = S * cap, ld if cap > 1 else ss
        else:
            ld, hs = self._rows(name, x, self.kv_heads, dt)
            rows = x.shape[0]
        _refuse(rows < 1, "%s is empty", name)
        return rows, ld, hs

    # ---- attention -----------------------------------------------------------------------------------------------------------------------
    def attend(self, q, k, v, q_start, k_start=None, slot=None, k_len=None, causal=True, max_k=None, lse=False, out=None):
        """softmax(scale * q k^T) v of B sequences of different lengths; returns o [Tq][heads][D] (or `out`; it must not overlap k or v).

        q [Tq][heads][D]; q_start [B + 1] int32 on the device, growing: sequence b owns the query rows q_start[b] .. q_start[b + 1] - 1 (n of them).
        k, v [Tk][kv_heads][D]: packed; sequence b's keys are the k_len[b] rows from k_start[b] on (both default to the queries' own rows).
        k, v [slots][cap][kv_heads][D]: a cache; its keys are the k_len[b] first rows of slot slot[b].
        causal: query i of n sees the keys j <= m - n + i of its m (a lone new token sees all of them).  Rows that see no key give 0; rows of no
        sequence are not written.  Starts, lengths and slots are int32 device tensors, clamped to the tensors by the kernel; max_k (host): an
        estimate of the longest m, which steers only how the work is split (default: a cache's cap, the number of packed key rows, or the average
        length where keys are the queries' own rows).  A caller who knows better should say so: a cache with much room to grow, one long sequence among
        short ones (up to twice the time otherwise).
        Scores, statistics and sums are fp32 and o is rounded once; 16-bit prompts also round each probability to the type for its product with v.
        lse=True: returns (o, lse [Tq][heads] float32), the log of each row's sum of exponentials (-inf where it sees no key)."""
        H, Hk, D, dt = self.heads, self.kv_heads, self.head_dim, getattr(q, "dtype", None)
        if dt not in _DTYPE:
            _refuse(True, "q is %s, wanted float32, float16 or bfloat16", dt)
        ldq, hsq = self._rows("q", q, H, dt)
        Tq = q.shape[0]
        if forward_ad._current_level >= 0:
            for name, x in (("q", q), ("k", k), ("v", v), ("out", out)):
                _no_gradient(name, x)
        B = q_start.numel() - 1 if isinstance(q_start, torch.Tensor) else -1
        _refuse(B < 0, "q_start: B + 1 values")
        qp = self._ints("q_start", q_start, B + 1)
        cap = ssk = ssv = sp = 0
        if isinstance(k, torch.Tensor) and k.dim() == 4:
            ssk, ldk, hsk = self._slots("k", k, dt)
            ssv, ldv, hsv = self._slots("v", v, dt)
            _refuse(slot is None or k_len is None or k_start is not None, "a cache [slots][cap] needs slot and k_len, and no k_start")
            sp = self._ints("slot", slot, B)
            longest = cap = k.shape[1]
        else:
            ldk, hsk = self._rows("k", k, Hk, dt)
            ldv, hsv = self._rows("v", v, Hk, dt)
            _refuse(slot is not None, "slot needs a cache [slots][cap][kv_heads][head_dim]")
            longest = k.shape[0]
            if k_start is not None:
                sp = self._ints("k_start", k_start, B)
            elif k_len is None and B > 1:
                longest = min(longest, Tq // B + 1)
        if k.shape != v.shape:
            _refuse(True, "k has shape %s, v %s", tuple(k.shape), tuple(v.shape))
        lp = self._ints("k_len", k_len, B) if k_len is not None else 0
        if out is None:
            out, ldo, hso = q.new_empty((Tq, H, D)), H * D, D
        else:
            ldo, hso = self._rows("out", out, H, dt, Tq)
        logs = torch.empty((Tq, H), dtype=torch.float32, device=self.device) if lse else None
        if Tq and B:
            slots, kp, vp = k.shape[0], k.data_ptr(), v.data_ptr()
            if not kp or not vp or not k.numel():               # nothing to read: every row of a sequence becomes 0
                slots = cap = sp = lp = 0
            if (Tq | slots | cap) >> 31:
                _refuse(True, "Tq=%d slots=%d cap=%d", Tq, slots, cap)
            if max_k is not None:
                longest = max(0, min(int(max_k), 0x7fffffff))
            head = (q.data_ptr(), kp, vp, out.data_ptr(), logs.data_ptr() if lse else 0, qp, sp, lp)
            longest = min(longest, 0x7fffffff)
            tail = (ldq, hsq, ldk, hsk, ldv, hsv, ldo, hso, ssk, ssv, Tq, B, slots, cap, H, Hk, D, _DTYPE[dt], bool(causal), longest, self.scale)
            ws, n = None, 0
            if longest > _SPLIT_KEYS:
                n = self.lib.value("deft_attn_ws_floats", _ATTN.pack(*head, 0, 0, *tail))
                if n:
                    ws = torch.empty(n, dtype=torch.float32, device=self.device)   # (stream-ordered: free for the next call once this one is queued)
            self._launch("deft_attn", _ATTN.pack(*head, ws.data_ptr() if n else 0, n, *tail))
        return (out, logs) if lse else out
