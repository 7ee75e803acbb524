"""Corners of deft_amd.attention, shared by the CPU (SIMT emulator) and the GPU tests.  References in 64 bits and tolerances: attention_checks.py."""
import math

import torch

import attention_checks as ac
from deft_amd.attention import AttentionPlan


def i32(device, *x):
    return torch.tensor(x, dtype=torch.int32, device=device)


def check_shared_key_rows(lib, device, dt, bad):
    """Key rows behind the last one are never used, also where the stride between rows is shorter than a row (one key, a cache of one row, expanded or
    sliding keys): an infinite or NaN value that IS visible comes back as it stands in the formula, not as 0 * inf of a row that is not there."""
    g = torch.Generator().manual_seed(3)
    D = 32
    plan = AttentionPlan(2, 1, D, device=device, lib=lib)
    q, k, v = ac.rand(g, dt, 5, 2, D).to(device), ac.rand(g, dt, 1, 1, D).to(device), ac.rand(g, dt, 1, 1, D).to(device)
    v[0, 0, 3] = bad

    def check(name, o, nq, keys, values, causal=True):
        want, _, A, mag = ac.ref_attend(q[:nq].cpu(), keys.cpu(), values.cpu(), plan.scale, causal)
        ac.assert_attended(name, o, want, A, mag, keys.shape[0], D, dt)

    check("one key", plan.attend(q[:1], k, v, i32(device, 0, 1)), 1, k, v)
    check("one key, not causal", plan.attend(q, k, v, i32(device, 0, 5), k_start=i32(device, 0), k_len=i32(device, 1), causal=False), 5, k, v, False)
    one = (i32(device, 0), i32(device, 1))
    check("cache of one row", plan.attend(q[:1], k[None], v[None], i32(device, 0, 1), slot=one[0], k_len=one[1]), 1, k, v)
    for causal in (True, False):
        ke, ve = k.expand(5, 1, D), v.expand(5, 1, D)
        check("expanded", plan.attend(q, ke, ve, i32(device, 0, 5), causal=causal), 5, ke, ve, causal)
    step = 16                                                        # rows that overlap: row r starts 16 elements behind row r - 1
    flat = ac.rand(g, dt, 5 * step + D).to(device)
    flat[4 * step + D - 1] = bad                                     # the last element of the last row of 5
    flat[4 * step + D] = float("nan")                                # what a sixth row would hold
    vs = flat.as_strided((5, 1, D), (step, step, 1))
    k5 = ac.rand(g, dt, 5, 1, D).to(device)
    for causal in (True, False):
        check("sliding", plan.attend(q, k5, vs, i32(device, 0, 5), causal=causal), 5, k5, vs, causal)


def check_unturned_elements(lib, device, dt, adjacent, norm):
    """Elements behind the 2 R first: as they were (normed where asked), whatever an element beside them holds."""
    g = torch.Generator().manual_seed(5)
    T, H, D, R = 7, 3, 64, 8
    q = ac.rand(g, dt, T, H, D)
    q[1, 0, 2 * R + 3], q[2, 1, D - 1], q[4, 2, D // 2 + 1] = float("inf"), float("-inf"), float("nan")
    pos = torch.arange(T, dtype=torch.int32).view(T, 1)
    plan = AttentionPlan(H, 1, D, axes=(R,), adjacent=adjacent, device=device, lib=lib)
    got, _ = (plan.norm_rotate if norm else plan.rotate)(q.to(device), None, pos.to(device))
    want, mag = ac.ref_rotate(q, pos, [10000.0 ** (-i / R) for i in range(R)], [0] * R, adjacent, norm=norm)
    got = got.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    if not norm:
        assert torch.equal(torch.nan_to_num(got[..., 2 * R:], 7.0), torch.nan_to_num(q[..., 2 * R:], 7.0))
    fine = torch.isfinite(want)
    ac.assert_rotated("finite", got[fine], want[fine], torch.nan_to_num(mag, 0, 0, 0)[fine], dt)


def check_norm_of_far_values(lib, device, dt, size, eps, T=6, H=5, D=64, R=24, inplace=False):
    """Heads whose squares leave fp32 (above about 1e19, below about 1e-19 where eps does not hold the mean up) are normed like any other; a head of zeros
    gives zeros, one with an infinity what the formula gives: 0 beside it, NaN in its place."""
    g = torch.Generator().manual_seed(6)
    q = (ac.rand(g, torch.float64, T, H, D) * size).to(dt)
    q[1, 2] = 1.0                                                     # an ordinary head among them
    if T > 6:
        q[6:, :H - 3] = ac.rand(g, dt, T - 6, H - 3, D)                # tokens whose last heads alone are far
    if eps > 0:
        q[2, 3] = 0.0
    q[3, 1, 7] = float("inf")
    pos = torch.arange(T, dtype=torch.int32).view(T, 1)
    plan = AttentionPlan(H, 1, D, axes=(R,), eps=eps, device=device, lib=lib)
    x = q.to(device, copy=True)
    got = plan.norm_rotate(x, None, pos.to(device), out=(x, None) if inplace else None)[0].cpu()
    want, mag = ac.ref_rotate(q, pos, [10000.0 ** (-i / R) for i in range(R)], [0] * R, False, norm=True, eps=eps)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert torch.isfinite(got[fine]).all()
    ac.assert_rotated("far values", got[fine], want[fine], mag[fine], dt)


def check_far_scores(lib, device, dt, size, H=2, Hk=1, D=32, nq=(3,), nk=(70,), causal=True, max_k=None, cache=None, equal=False):
    """Finite scores of any size: the softmax of the scores as they are (`equal`: all the same, so that o is the mean of the values and lse the score plus
    log m), never 0 or NaN because they left the range of an exponential.  Every score is exact in fp32 (few bits, one product), so it is the softmax that is
    tested: where the scores differ, they differ by so much that the largest alone counts."""
    g = torch.Generator().manual_seed(7)
    b = ac.make_batch(dt, list(nq), list(nk), H, Hk, D, device, cache)
    scale = 1.0 if abs(size) > 1e37 else 0.25                        # (q . k itself stays in fp32)
    plan = AttentionPlan(H, Hk, D, scale=scale, device=device, lib=lib)
    root = 2.0 ** (round(math.log2(abs(size) / scale)) // 2)
    q = torch.zeros(b["q"].shape, dtype=torch.float64)
    q[..., 0] = root                                                 # a score is scale * root * k[..., 0]
    keys = []
    for i, n in enumerate(nk):
        k, v = (torch.zeros(n, Hk, D, dtype=torch.float64), ac.rand(g, dt, n, Hk, D))
        k[..., 0] = size / scale / root
        if not equal:
            k[..., 0] *= (1 + torch.randperm(n, generator=g)[:, None] / 128)       # (8 bits: exact in every type)
        k = k.to(dt)
        keys.append((k, v))
        if cache:
            b["k"][b["slot"][i].long(), :n], b["v"][b["slot"][i].long(), :n] = k.to(device), v.to(device)
        else:
            at = sum(nk[:i])
            b["k"][at:at + n], b["v"][at:at + n] = k.to(device), v.to(device)
    q = q.to(dt).to(device)
    kw = {n: b[n] for n in ("k_start", "slot", "k_len") if n in b}
    o, lse = plan.attend(q, b["k"], b["v"], b["q_start"], causal=causal, max_k=max_k, lse=True, **kw)
    for i in range(len(nq)):
        s = slice(b["starts"][i], b["starts"][i + 1])
        want, wl, A, mag = ac.ref_attend(q[s].cpu(), *keys[i], plan.scale, causal)
        assert torch.isfinite(want).all() and torch.isfinite(wl).all()
        ac.assert_attended("scores of %g, sequence %d" % (size, i), o[s], want, A, torch.zeros_like(mag), nk[i], D, dt)
        # lse: the largest score rounded to fp32 before and after the factor 2 ln 2, and 12 u + m / 2 u of the sum
        assert bool(((lse[s].double().cpu() - wl).abs() <= 4 * ac.U * wl.abs() + 12 * ac.U + nk[i] * ac.U / 2).all()), "lse of scores of %g" % size


def check_starts_that_do_not_grow(lib, device):
    """q_start that does not grow, keys split: a row of the output is left as it was or is what one of the sequences that name it gives -- never what stood in
    the workspace (the caller has it hold NaN)."""
    g = torch.Generator().manual_seed(9)
    q, k = ac.rand(g, torch.float32, 4, 2, 32).to(device), ac.rand(g, torch.float32, 900, 1, 32).to(device)
    plan = AttentionPlan(2, 1, 32, device=device, lib=lib)
    ks, kl = i32(device, 0, 300, 900 - 270), i32(device, 300, 280, 270)
    for starts in ((0, 4, 2, 4), (3, 1, 0, 4), (-7, 2, 99, 3), (4, 0, 4, 0), (0, 3, 1, 4), (2, 4, 0, 2)):
        out = torch.full((4, 2, 32), 5.0, device=device)
        o = plan.attend(q, k, k, i32(device, *starts), k_start=ks, k_len=kl, max_k=700, out=out)
        cut = [min(max(s, 0), 4) for s in starts]
        for t in range(4):
            may = [torch.full((2, 32), 5.0, dtype=torch.float64)]
            tol = [torch.zeros(2, 32, dtype=torch.float64)]
            for b in range(3):
                n = cut[b + 1] - cut[b]
                if cut[b] <= t < cut[b + 1]:
                    a, m = int(ks[b]), int(kl[b])
                    want, _, A, mag = ac.ref_attend(q[cut[b]:cut[b] + n].cpu(), k[a:a + m].cpu(), k[a:a + m].cpu(), plan.scale, True)
                    may.append(want[t - cut[b]])
                    tol.append((2 * (2 * 36 * ac.U * mag[t - cut[b]] + 8 * ac.U + m * ac.U / 2))[:, None] * A[t - cut[b]] + ac.U * want[t - cut[b]].abs())
            got = o[t].double().cpu()
            assert any(bool(((got - w).abs() <= e).all()) for w, e in zip(may, tol)), "starts %s, row %d" % (starts, t)


def check_masked_values(lib, device, dt, D, bad, nq, nk, max_k, cache="slots"):
    """Infinities and NaN in the last keys and values of every sequence (and in all memory behind them): rows that do not see them are as close to the formula
    as ever, rows that do come out as the formula says."""
    def spoil(b):
        for i, (k, v) in enumerate(b["keys"]):
            m = k.shape[0]
            k[-1], v[-1], v[-2, :, ::3] = bad, bad, bad
            if cache:
                s = int(b["slot"][i])
                b["k"][s, :m], b["v"][s, :m] = k.to(device), v.to(device)
            else:
                at = sum(nk[:i])
                b["k"][at:at + m], b["v"][at:at + m] = k.to(device), v.to(device)

    b = ac.make_batch(dt, list(nq), list(nk), 2, 1, D, device, cache, seed=2, poison=bool(cache))
    spoil(b)
    plan = AttentionPlan(2, 1, D, device=device, lib=lib)
    o = plan.attend(b["q"], b["k"], b["v"], b["q_start"], max_k=max_k, **{n: b[n] for n in ("k_start", "slot", "k_len") if n in b})
    for i, (n, m) in enumerate(zip(nq, nk)):
        got = o[b["starts"][i]:b["starts"][i + 1]]
        want, _, A, mag = ac.ref_attend(b["queries"][i], *b["keys"][i], plan.scale, True)
        ac.assert_attended("sequence %d, early rows" % i, got[:n - 2], want[:n - 2], A[:n - 2], mag[:n - 2], m, D, dt)
        # the last but one sees the spoiled values of its last key (every third column); the last one sees a spoiled key
        assert not torch.isfinite(got[n - 2, :, ::3]).any()
        keep = [c for c in range(D) if c % 3]
        ac.assert_attended("sequence %d, last row but one" % i, got[n - 2:n - 1, :, keep], want[n - 2:n - 1, :, keep], A[n - 2:n - 1, :, keep], mag[n - 2:n - 1], m, D, dt)
        assert not torch.isfinite(got[n - 1]).all()


def check_seen_infinities(lib, device, dt, D, nq, nk, max_k, cache="slots"):
    """Infinities and NaN among the values every row sees: they come out in their columns as the formula says, whatever probability they meet; the other
    columns are as close as ever."""
    inf = float("inf")
    b = ac.make_batch(dt, list(nq), list(nk), 2, 1, D, device, cache, seed=4, poison=bool(cache))
    for i, (k, v) in enumerate(b["keys"]):
        m = k.shape[0]
        v[0, :, 0], v[0, :, 1], v[0, :, 2], v[1, :, 2], v[0, :, 3] = inf, -inf, inf, -inf, float("nan")
        k[0] *= 3.0                                                    # (some rows hardly look at it)
        if cache:
            s = int(b["slot"][i])
            b["k"][s, :m], b["v"][s, :m] = k.to(device), v.to(device)
        else:
            at = sum(nk[:i])
            b["k"][at:at + m], b["v"][at:at + m] = k.to(device), v.to(device)
    plan = AttentionPlan(2, 1, D, device=device, lib=lib)
    o = plan.attend(b["q"], b["k"], b["v"], b["q_start"], max_k=max_k, causal=False, **{n: b[n] for n in ("k_start", "slot", "k_len") if n in b})
    for i, m in enumerate(nk):
        want, _, A, mag = ac.ref_attend(b["queries"][i], *b["keys"][i], plan.scale, False)
        assert torch.equal(want[:, :, 0], torch.full_like(want[:, :, 0], inf)) and torch.isnan(want[:, :, 2:4]).all()
        ac.assert_attended("sequence %d" % i, o[b["starts"][i]:b["starts"][i + 1]], want, A, mag, m, D, dt)


def check_two_piece_steps(lib, device, dt, D, nq, nk, max_k):
    """The step kernel's products take a probability whole (two pieces: 2^-16 relative and better): beyond the output's own rounding its error is fp32's."""
    g = torch.Generator().manual_seed(8)
    b = ac.make_batch(dt, list(nq), list(nk), 6, 2, D, device, "slots", seed=8)
    plan = AttentionPlan(6, 2, D, device=device, lib=lib)
    o = plan.attend(b["q"], b["k"], b["v"], b["q_start"], slot=b["slot"], k_len=b["k_len"], max_k=max_k)
    for i, m in enumerate(nk):
        want, _, A, mag = ac.ref_attend(b["queries"][i], *b["keys"][i], plan.scale, True)
        # bf16: the rest is rounded to half a step of a number below half a step (2^-8 2^-8), fp16 likewise (2^-22) as far as its subnormals reach (2^-25 of
        # a largest P of 2^6)
        fine = 2.0 ** -16 if dt == torch.bfloat16 else 2.0 ** -22
        tol = (2 * (2 * (D + 4) * ac.U * mag + 8 * ac.U + m * ac.U / 2) + fine)[..., None] * A + ac.half(dt) * want.abs() + ac.tiny(dt) + (m * 2.0 ** -31 * 8 if dt == torch.float16 else 0)
        err = (o[b["starts"][i]:b["starts"][i + 1]].double().cpu() - want).abs()
        assert bool((err <= tol).all()), "sequence %d: %.3g of its tolerance" % (i, float((err / tol).max()))


def check_in_place(lib, device, dt):
    """attend may write onto its queries: every kernel reads a tile's rows before it writes them."""
    for nq, nk, max_k in (((1, 1, 5), (60, 31, 5), None), ((1, 2), (900, 255), None), ((1, 2), (300, 255), 200), ((150, 70), (150, 70), None), ((150,), (700,), 700)):
        b = ac.make_batch(dt, list(nq), list(nk), 6, 2, 64, device, "slots", seed=11, poison=True)
        plan = AttentionPlan(6, 2, 64, device=device, lib=lib)
        kw = dict(slot=b["slot"], k_len=b["k_len"], max_k=max_k)
        want = plan.attend(b["q"], b["k"], b["v"], b["q_start"], **kw)
        got = plan.attend(b["q"], b["k"], b["v"], b["q_start"], out=b["q"], **kw)
        assert got is b["q"] and torch.equal(got, want)


def check_shared_keys(lib, device, dt):
    """Sequences that read the same keys: one slot for several, windows of the packed rows that overlap."""
    g = torch.Generator().manual_seed(12)
    H, Hk, D = 4, 2, 32
    plan = AttentionPlan(H, Hk, D, device=device, lib=lib)
    nq, slots, nk = (1, 3, 1, 40), (1, 1, 0, 1), (50, 50, 7, 33)
    qs = [0]
    for n in nq:
        qs.append(qs[-1] + n)
    q, k, v = ac.rand(g, dt, qs[-1], H, D).to(device), ac.rand(g, dt, 2, 60, Hk, D).to(device), ac.rand(g, dt, 2, 60, Hk, D).to(device)
    o = plan.attend(q, k, v, i32(device, *qs), slot=i32(device, *slots), k_len=i32(device, *nk))
    at = (0, 20, 20, 5)
    kp, vp = k.view(120, Hk, D), v.view(120, Hk, D)
    op = plan.attend(q, kp, vp, i32(device, *qs), k_start=i32(device, *at), k_len=i32(device, *nk))
    for i, n in enumerate(nq):
        s = slice(qs[i], qs[i + 1])
        for name, got, keys, vals in (("slot", o, k[slots[i], :nk[i]], v[slots[i], :nk[i]]), ("window", op, kp[at[i]:at[i] + nk[i]], vp[at[i]:at[i] + nk[i]])):
            want, _, A, mag = ac.ref_attend(q[s].cpu(), keys.cpu(), vals.cpu(), plan.scale, True)
            ac.assert_attended("%s %d" % (name, i), got[s], want, A, mag, nk[i], D, dt)


def check_many_sequences(lib, device, dt, B):
    """One token a sequence, thousands of them: each sees itself alone and gives its value back (P = 1 up to the fma's last step, twice rounded)."""
    g = torch.Generator().manual_seed(13)
    plan = AttentionPlan(2, 1, 32, device=device, lib=lib)
    q, k, v = ac.rand(g, dt, B, 2, 32).to(device), ac.rand(g, dt, B, 1, 32).to(device), ac.rand(g, dt, B, 1, 32).to(device)
    o, lse = plan.attend(q, k, v, torch.arange(B + 1, dtype=torch.int32, device=device), lse=True)
    want = v.expand(B, 2, 32).double()
    assert bool(((o.double() - want).abs() <= (ac.half(dt) + 4 * ac.U) * want.abs() + ac.tiny(dt)).all())
    s = (q.double() * k.double()).sum(-1) * plan.scale
    mag = (q.double() * k.double()).abs().sum(-1) * plan.scale
    assert bool(((lse.double() - s).abs() <= 2 * 36 * ac.U * mag + 12 * ac.U).all())


def check_far_scores_beside_masked_values(lib, device, dt, max_k):
    """Both reasons for a second pass in one tile: scores beyond the reference's range, infinities behind the diagonal."""
    g = torch.Generator().manual_seed(14)
    n, D = 70, 64
    plan = AttentionPlan(2, 1, D, scale=0.25, device=device, lib=lib)
    q, k, v = torch.zeros(n, 2, D, dtype=torch.float64), torch.zeros(n, 1, D, dtype=torch.float64), ac.rand(g, dt, n, 1, D)
    q[..., 0], k[..., 0] = 2.0 ** 50, -2.0 ** 50 * (1 + torch.randperm(n, generator=g)[:, None] / 128)
    q, k = q.to(dt), k.to(dt)
    v[-1], v[-2, :, ::3] = float("nan"), float("inf")
    o = plan.attend(q.to(device), k.to(device), v.to(device), i32(device, 0, n), max_k=max_k)
    want, _, A, mag = ac.ref_attend(q, k, v, plan.scale, True)
    ac.assert_attended("rows", o[:n - 2], want[:n - 2], A[:n - 2], torch.zeros_like(mag)[:n - 2], n, D, dt)
    assert not torch.isfinite(o[n - 1]).any() and not torch.isfinite(o[n - 2, :, ::3]).any()
