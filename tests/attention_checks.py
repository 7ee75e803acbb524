"""Checks of deft_amd.attention against plain implementations in 64 bits, shared by the CPU (SIMT emulator) and the GPU tests.

u = 2^-24 is half an fp32 step; h(t) = torch.finfo(t).eps / 2 half a step of the element type, both relative to the value.
"""
import math

import torch

from deft_amd.attention import AttentionPlan

U = 2.0 ** -24


def half(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Half the smallest step of the type: what rounding loses below its normal range."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def rand(g, dt, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float64).to(dt)


# ---- rotary positions and norms ------------------------------------------------------------------------------------------------------------

def ref_rotate(x, pos, freq, axis, adjacent, inverse=False, norm=False, w=None, eps=1e-6):
    """(result, |x| + |y| of each element's pair) in 64 bits on the CPU."""
    y = x.double().cpu()
    if norm:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if w is not None:
            y = y * w.double().cpu()
    R = len(freq)
    ang = pos.double().cpu()[:, axis] * torch.as_tensor(freq, dtype=torch.float64)
    if inverse:
        ang = -ang
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    out, mag = y.clone(), y.abs().clone()
    i0 = torch.arange(0, 2 * R, 2) if adjacent else torch.arange(R)
    i1 = i0 + 1 if adjacent else i0 + R
    a, b = y[..., i0], y[..., i1]
    out[..., i0], out[..., i1] = a * c - b * s, b * c + a * s
    mag[..., i0] = mag[..., i1] = a.abs() + b.abs()
    return out, mag


def assert_rotated(name, got, want, mag, dt):
    # fp32 part: the norm's sum of <= 256 squares is a chain of <= 16 fma and <= 5 butterfly adds (21 u, halved by the root), root, two divisions
    # and two products (5 u): 16 u; sine and cosine 2 u absolute; products and sum of the rotation 3 u: 21 u of |x| + |y|, 24 taken
    tol = half(dt) * want.abs() + 24 * U * mag * (1 + half(dt)) + tiny(dt)
    err = (got.double().cpu() - want).abs()
    bad = err > tol
    assert not bad.any(), "%s: %d of %d off, worst %.3g of its tolerance" % (name, int(bad.sum()), bad.numel(), float((err / tol).max()))


def check_rotary(lib, device, dt, T, H, Hk, D, axes, adjacent=False, frac=False, norm=False, cache=None, inverse=False, inplace=False, far=False, seed=0,
                 weights=True, k_none=False):
    """cache: None, "rows" ([rows][Hk][D]) or "slots" ([slots][cap][Hk][D])."""
    g = torch.Generator().manual_seed(seed)
    R = sum(axes)
    buf = rand(g, dt, T, H + 2 * Hk, D).to(device)
    q, k, v = buf[:, :H], buf[:, H:H + Hk], buf[:, H + Hk:]
    pos = torch.rand(T, len(axes), generator=g, dtype=torch.float64) * (1e6 if far else 1000.0) - (0.0 if far else 300.0)
    pos = (pos.float() if frac else pos.to(torch.int32)).to(device)
    qw, kw = (1 + 0.3 * torch.randn(D, generator=g) for _ in range(2)) if weights else (None, None)
    plan = AttentionPlan(H, Hk, D, axes=axes, adjacent=adjacent, q_weight=qw, k_weight=kw, device=device, lib=lib)
    axis = [a for a, n in enumerate(axes) for _ in range(n)]
    freq = [10000.0 ** (-i / R) for i in range(R)]
    wq, mq = ref_rotate(q, pos, freq, axis, adjacent, inverse, norm, qw)
    wk, mk = ref_rotate(k, pos, freq, axis, adjacent, inverse, norm, kw)
    before = buf.clone()
    kw_ = {} if norm else {"inverse": inverse}
    fn = plan.norm_rotate if norm else plan.rotate
    if cache:
        S, cap = 3, T // 3 + 4
        rows = S * cap
        kc, vc = (rand(g, dt, S, cap, Hk, D).to(device) for _ in range(2))
        if cache == "rows":
            kc, vc = kc.view(rows, Hk, D), vc.view(rows, Hk, D)
        k0, v0 = kc.clone().view(rows, Hk, D), vc.clone().view(rows, Hk, D)
        row = torch.randperm(rows, generator=g)[:T].to(torch.int32)
        if T > 2:
            row[1], row[T - 1] = -1, rows                     # outside: not written
        got_q, got_k = fn(q, k, pos, v=v, cache=(kc, vc), row=row.to(device), **kw_)
        assert got_k is kc
        assert_rotated("q", got_q, wq, mq, dt)
        on = (row >= 0) & (row < rows)
        r = row[on].long()
        assert_rotated("k rows", kc.view(rows, Hk, D).cpu()[r], wk[on], mk[on], dt)
        assert torch.equal(vc.view(rows, Hk, D).cpu()[r], v.cpu()[on])
        rest = torch.ones(rows, dtype=torch.bool)
        rest[r] = False
        assert torch.equal(kc.view(rows, Hk, D).cpu()[rest], k0.cpu()[rest]) and torch.equal(vc.view(rows, Hk, D).cpu()[rest], v0.cpu()[rest])
    elif inplace:
        got_q, got_k = fn(q, k, pos, out=(q, k), **kw_)
        assert got_q is q and got_k is k
        assert_rotated("q", q, wq, mq, dt)
        assert_rotated("k", k, wk, mk, dt)
        assert torch.equal(buf[:, H + Hk:], before[:, H + Hk:])
        return
    else:
        got_q, got_k = fn(q, None if k_none else k, pos, **kw_)
        assert_rotated("q", got_q, wq, mq, dt)
        if k_none:
            assert got_k is None
        else:
            assert_rotated("k", got_k, wk, mk, dt)
    assert torch.equal(buf, before)


# ---- attention -----------------------------------------------------------------------------------------------------------------------------

def ref_attend(q, k, v, scale, causal):
    """One sequence, 64 bits: q [n][H][D], k, v [m][Hk][D] -> o [n][H][D], lse [n][H], sum_j p |v| / L, max |q||k| sums.  A masked key takes no part
    whatever it holds: only the visible keys of a row are looked at."""
    n, H, D = q.shape
    m, Hk = k.shape[0], k.shape[1]
    G = H // Hk
    o, A = torch.zeros(n, H, D, dtype=torch.float64), torch.zeros(n, H, D, dtype=torch.float64)
    lse, mag = torch.full((n, H), -math.inf, dtype=torch.float64), torch.zeros(n, H, dtype=torch.float64)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    for h in range(H):
        kh, vh = k[:, h // G], v[:, h // G]
        if m == 0:
            continue
        s = q[:, h] @ kh.T * scale
        a = q[:, h].abs() @ kh.abs().T * scale
        vis = torch.ones(n, m, dtype=torch.bool)
        if causal:
            vis = torch.arange(m)[None] <= (m - n + torch.arange(n))[:, None]
        some = vis.any(-1)
        s = s.masked_fill(~vis, -math.inf)
        mag[:, h] = a.masked_fill(~vis, 0).amax(-1)
        M = s.amax(-1, keepdim=True)
        p = torch.where(vis, torch.exp(s - M), 0.0)
        L = p.sum(-1, keepdim=True)
        if torch.isfinite(vh).all():
            o[:, h] = torch.where(some[:, None], p @ vh / L, 0.0)
        else:
            for i in range(n):
                if some[i]:
                    o[i, h] = (p[i, vis[i]][:, None] * vh[vis[i]]).sum(0) / L[i]
        A[:, h] = torch.where(some[:, None], p @ torch.nan_to_num(vh.abs(), 0, 0, 0) / L, 0.0)
        lse[:, h] = torch.where(some, (M + L.log())[:, 0], -math.inf)
    return o, lse, A, mag


def assert_attended(name, got, want, A, mag, m, D, dt):
    """A = sum_j p_j |v_j| / L.  A probability is off by its score's error -- (D + 2) u of mag = scale sum |q k|, twice that for the difference to
    the maximum and its scaling to base 2 -- plus 8 u for the exponential; the sums of m terms by m / 2 u more (pairwise blocks do better); both for
    the numerator and the denominator.  16-bit types round each probability once more (h, numerator only), fp16 ones not below 2^-31 of the largest
    (subnormal: 2^-25 of a maximum kept at 2^6 or above); the result is rounded once."""
    fp32 = 2 * (2 * (D + 4) * U * mag + 8 * U + m * U / 2)
    rel = fp32 if dt == torch.float32 else fp32 + half(dt) * (1 + half(dt))
    tol = rel[..., None] * A + half(dt) * want.abs() + tiny(dt)
    if dt == torch.float16:
        tol = tol + m * 2.0 ** -31 * 8
    got = got.double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name + ": NaN where it should not be, or none where it should"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), name + ": infinities differ"
    err = (got - want)[fine].abs()
    bad = err > tol[fine]
    assert not bad.any(), "%s: %d of %d off, worst %.3g of its tolerance" % (name, int(bad.sum()), bad.numel(), float((err / tol[fine]).max()))


def make_batch(dt, nq, nk, H, Hk, D, device, cache=None, seed=0, poison=False, gap=0, head_major=False):
    """Tensors of a batch.  cache None: packed, keys of sequence b behind each other (own k_start when they differ from the queries); "slots": a cache.
    poison: everything no sequence may read is NaN or infinite.  gap: rows in front of the first and behind the last sequence."""
    g = torch.Generator().manual_seed(seed)
    B, Tq = len(nq), sum(nq) + 2 * gap
    bad = float("nan") if poison else 0.5
    q = rand(g, dt, Tq, H, D)
    starts = [gap]
    for n in nq:
        starts.append(starts[-1] + n)
    b = {"q_start": torch.tensor(starts, dtype=torch.int32, device=device)}
    if cache:
        S, cap = B + 2, max(list(nk) + [1]) + 3
        k, v = rand(g, dt, S, cap, Hk, D), rand(g, dt, S, cap, Hk, D)
        slot = torch.randperm(S, generator=g)[:B]
        keep = torch.zeros(S, cap, dtype=torch.bool)
        for i in range(B):
            keep[slot[i], :nk[i]] = True
        k[~keep], v[~keep] = bad, (float("inf") if poison else 0.5)
        b["slot"], b["k_len"] = slot.to(torch.int32).to(device), torch.tensor(nk, dtype=torch.int32, device=device)
        b["keys"] = [(k[slot[i], :nk[i]], v[slot[i], :nk[i]]) for i in range(B)]
    else:
        ks = [gap]
        for n in nk:
            ks.append(ks[-1] + n)
        k, v = rand(g, dt, ks[-1] + gap, Hk, D), rand(g, dt, ks[-1] + gap, Hk, D)
        if gap:
            for x in (k, v):
                x[:gap], x[ks[-1]:] = bad, bad
        if list(nk) != list(nq):
            b["k_start"], b["k_len"] = (torch.tensor(x, dtype=torch.int32, device=device) for x in (ks[:-1], list(nk)))
        b["keys"] = [(k[ks[i]:ks[i + 1]], v[ks[i]:ks[i + 1]]) for i in range(B)]
    if head_major and not cache:                                      # [head][token][D] storage
        k, v = (x.transpose(0, 1).contiguous().to(device).transpose(0, 1) for x in (k, v))
    b["q"], b["k"], b["v"] = q.to(device), k.to(device), v.to(device)
    b["queries"] = [q[starts[i]:starts[i + 1]] for i in range(B)]
    b["starts"] = starts
    return b


def check_attend(lib, device, dt, nq, nk, H, Hk, D, causal=True, cache=None, seed=0, poison=False, gap=0, head_major=False, max_k=None, mutate=None, scale=None):
    b = make_batch(dt, nq, nk, H, Hk, D, device, cache, seed, poison, gap, head_major)
    if mutate is not None:
        mutate(b)
    plan = AttentionPlan(H, Hk, D, scale=scale, device=device, lib=lib)
    out = torch.full_like(b["q"], 7.0).contiguous()
    kw = {n: b[n] for n in ("k_start", "slot", "k_len") if n in b}
    o, lse = plan.attend(b["q"], b["k"], b["v"], b["q_start"], causal=causal, max_k=max_k, lse=True, out=out, **kw)
    assert o is out
    for i in range(len(nq)):
        s0, s1 = b["starts"][i], b["starts"][i + 1]
        want, wl, A, mag = ref_attend(b["queries"][i], *b["keys"][i], plan.scale, causal)
        assert_attended("sequence %d" % i, o[s0:s1], want, A, mag, nk[i], D, dt)
        fin = torch.isfinite(wl)
        gl = lse[s0:s1].double().cpu()
        assert torch.equal(gl[~fin & ~wl.isnan()], wl[~fin & ~wl.isnan()]), "lse of sequence %d" % i
        lt = 2 * (D + 4) * U * mag + 12 * U + nk[i] * U / 2 + 2 * U * wl.abs()
        assert bool(((gl - wl).abs() <= lt)[fin].all()), "lse of sequence %d: off by %g" % (i, float((gl - wl)[fin].abs().max()))
    rest = torch.ones(o.shape[0], dtype=torch.bool)
    rest[b["starts"][0]:b["starts"][-1]] = False
    assert (o.cpu()[rest] == 7.0).all()                              # rows of no sequence: as they were
    return o
