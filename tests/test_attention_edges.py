"""-m "not gpu": corners of the attention-layer operators through the SIMT emulator; the checks themselves are in tests/attention_edges.py."""
import pytest
import torch

import attention_edges as ae

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_key_rows_that_share_memory(emu_lib, dt, bad):
    ae.check_shared_key_rows(emu_lib, "cpu", dt, bad)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_unturned_elements(emu_lib, dt, adjacent, norm):
    ae.check_unturned_elements(emu_lib, "cpu", dt, adjacent, norm)


@pytest.mark.parametrize("dt,size,eps", [(F32, 1e25, 1e-6), (BF16, 1e30, 1e-6), (F32, 3e37, 0.0), (F32, 1e-25, 0.0), (BF16, 1e-30, 0.0), (F32, 1e-20, 1e-38), (F16, 1e-5, 0.0),
                                         (F32, 1e-30, 1e-6), (BF16, 1e19, 1e-6)])
def test_norm_of_far_values(emu_lib, dt, size, eps):
    ae.check_norm_of_far_values(emu_lib, "cpu", dt, size, eps)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_norm_of_far_values_among_others(emu_lib, dt):
    """Waves of several passes, a far head in the last: what the earlier passes have written in place is not read again."""
    ae.check_norm_of_far_values(emu_lib, "cpu", dt, 1e25, 1e-6, T=1400, H=80 if dt == F32 else 160, D=32, R=16, inplace=True)


FAR = [dict(size=s, equal=e) for s in (1e8, -1e8, 1e12, -1e12, 1e30, -1e30, 2e38, -2e38, -3e38, 3e38) for e in (True, False) if e or abs(s) < 1e38]


@pytest.mark.parametrize("kw", FAR)
@pytest.mark.parametrize("dt", [F32, BF16])
def test_far_scores(emu_lib, dt, kw):
    ae.check_far_scores(emu_lib, "cpu", dt, **kw)                                                    # one-wave step kernel
    ae.check_far_scores(emu_lib, "cpu", dt, nq=(2, 3), nk=(300, 40), max_k=300, cache="slots", **kw)     # four waves
    ae.check_far_scores(emu_lib, "cpu", dt, nq=(1,), nk=(600,), max_k=600, cache="slots", **kw)          # keys split
    ae.check_far_scores(emu_lib, "cpu", dt, nq=(80,), nk=(90,), **kw)                                # prompt kernel
    ae.check_far_scores(emu_lib, "cpu", dt, nq=(70,), nk=(600,), max_k=1100, causal=False, **kw)     # prompt, split


@pytest.mark.parametrize("size", [1e5, -1e5, 1e8, -1e8])
def test_far_scores_fp16(emu_lib, size):
    for equal in (True, False):
        ae.check_far_scores(emu_lib, "cpu", F16, size, equal=equal)
        ae.check_far_scores(emu_lib, "cpu", F16, size, nq=(80,), nk=(90,), equal=equal)


def test_starts_that_do_not_grow(emu_lib, monkeypatch):
    empty = torch.empty                                              # host memory comes back as zeros or as anything: here the workspace is NaN
    monkeypatch.setattr(torch, "empty", lambda *a, **k: empty(*a, **k).fill_(float("nan")) if k.get("dtype") is torch.float32 else empty(*a, **k))
    ae.check_starts_that_do_not_grow(emu_lib, "cpu")


def test_every_gradient_is_refused(emu_lib):
    """Weights, frequencies and positions that need a gradient, and forward-mode tangents, are refused like q, k, v: nothing drops out silently."""
    from deft_amd.attention import AttentionPlan
    from deft_amd.hiplib import DeftHipError
    import torch.autograd.forward_ad as fw
    P = lambda **kw: AttentionPlan(2, 1, 32, axes=(16,), device="cpu", lib=emu_lib, **kw)  # noqa: E731
    w = torch.nn.Parameter(torch.ones(32))
    f = torch.ones(16, dtype=torch.float64, requires_grad=True)
    for kw in (dict(q_weight=w), dict(k_weight=w), dict(freq=f)):
        with pytest.raises(DeftHipError, match="forward only"):
            P(**kw)
        with torch.no_grad():
            P(**kw)
    plan = P(q_weight=w.detach())
    q, k, qs = torch.ones(2, 2, 32), torch.ones(2, 1, 32), torch.tensor([0, 2], dtype=torch.int32)
    pos = torch.ones(2, 1, requires_grad=True)
    with pytest.raises(DeftHipError, match="forward only"):
        plan.rotate(q, k, pos)
    with torch.no_grad():
        plan.rotate(q, k, pos)
    pos = pos.detach()
    with fw.dual_level():
        d = lambda x: fw.make_dual(x, torch.ones_like(x))  # noqa: E731
        plan.rotate(q, k, pos), plan.attend(q, k, k, qs)                       # no tangent among them
        for call in (lambda: plan.rotate(d(q), k, pos), lambda: plan.rotate(q, d(k), pos), lambda: plan.norm_rotate(q, k, d(pos)), lambda: plan.attend(d(q), k, k, qs),
                     lambda: plan.attend(q, d(k), k, qs), lambda: plan.attend(q, k, d(k), qs), lambda: P(q_weight=d(torch.ones(32)))):
            with pytest.raises(DeftHipError, match="forward only"):
                call()


def test_weights_are_copied(emu_lib):
    from deft_amd.attention import AttentionPlan
    w = torch.full((32,), 2.0)
    plan = AttentionPlan(2, 1, 32, axes=(16,), q_weight=w, device="cpu", lib=emu_lib)
    q, pos = torch.ones(1, 2, 32), torch.zeros(1, 1, dtype=torch.int32)
    a = plan.norm_rotate(q, None, pos)[0]
    w.zero_()
    assert torch.equal(plan.norm_rotate(q, None, pos)[0], a) and a.abs().max() > 1


def test_plans_no_call_could_use_are_refused(emu_lib):
    """What no call of a plan could take is refused when the plan is made; what one operator or type alone takes, at the call that does not."""
    from deft_amd.attention import AttentionPlan
    from deft_amd.hiplib import DeftHipError
    P = lambda **kw: AttentionPlan(**{**dict(heads=4, kv_heads=2, head_dim=64, device="cpu", lib=emu_lib), **kw})  # noqa: E731
    for kw, word in [(dict(axes=(13,)), "R=13 pairs"), (dict(head_dim=33), "D=33"), (dict(head_dim=0), "D=0"), (dict(head_dim=264), "D=264"), (dict(scale=0.0), "scale=0"),
                     (dict(scale=-1.0), "scale=-1"), (dict(scale=float("nan")), "scale=nan"), (dict(scale=float("inf")), "scale=inf"), (dict(eps=-1e-6), "eps="),
                     (dict(eps=float("nan")), "eps=nan"), (dict(heads=8192, kv_heads=8192), "4096"), (dict(axes=(4,) * 9, head_dim=128), "9 axes"), (dict(scale=1e-39), "scale=1e-39")]:
        with pytest.raises(DeftHipError, match=word):
            P(**kw)
    for kw in (dict(head_dim=40, axes=(8, 12)), dict(head_dim=256, axes=(128,)), dict(axes=(4,)), dict(axes=(4,) * 8), dict(scale=2.0 ** -126), dict(eps=0.0)):
        P(**kw)


def test_an_older_library_says_rebuild(monkeypatch):
    """A library without an entry point of this package is refused with the advice to rebuild, not with an AttributeError."""
    import ctypes as C
    from deft_amd import build, hiplib
    so = build.build(force=False, verbose=False)
    monkeypatch.setitem(hiplib._SIGS, "deft_not_yet_there", (C.c_int, []))
    with pytest.raises(hiplib.DeftHipError, match="deft_not_yet_there.*rebuild"):
        hiplib.HipLib(so)


def test_sizes_beyond_the_descriptor_are_refused(emu_lib):
    """Token, row and slot counts past what a launch or the descriptor holds: the documented error, whatever the count (views of one token cost no memory)."""
    import ctypes as C
    from deft_amd.attention import AttentionPlan
    from deft_amd.hiplib import DeftHipError, RotaryDesc
    plan = AttentionPlan(1, 1, 32, axes=(16,), device="cpu", lib=emu_lib)
    one = torch.zeros(1, 1, 32)
    pos, qs, s1 = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for T in ((1 << 30) + 1, 1 << 31, 1 << 33):
        with pytest.raises(DeftHipError, match="tokens"):
            plan.rotate(one.expand(T, 1, 32), None, pos)
    for n in ((1 << 30) + 1, 1 << 31, 1 << 33):
        many = one.expand(n, 1, 32)
        with pytest.raises(DeftHipError, match="slots="):
            plan.attend(one, many, many, qs)
        with pytest.raises(DeftHipError, match="cap="):
            plan.attend(one, many[None], many[None], qs, slot=s1, k_len=s1)
        with pytest.raises(DeftHipError, match="Tq="):
            plan.attend(many, one, one, qs, out=torch.zeros(1, 1, 32).expand(n, 1, 32))
    d, buf = RotaryDesc(), torch.zeros(64)
    for f in ("q", "q_out", "pos", "freq", "axis"):
        setattr(d, f, buf.data_ptr() + (-buf.data_ptr()) % 16)
    d.T, d.Hq, d.Hk, d.D, d.R, d.A, d.ldq, d.hsq, d.ldqo, d.hsqo = (1 << 26) - 3, 64, 1, 8, 4, 1, 512, 8, 512, 8      # 64 heads of one lane: a wave a token
    with pytest.raises(DeftHipError, match="T=67108861"):
        emu_lib.call("deft_rotary", C.byref(d), None)


def test_the_twins_forward(emu_lib):
    """The `_p3` names of the operators without pieces: the same results, the refusal's text in their own set; their kernels are in the library once."""
    import os
    import subprocess
    from deft_amd import build
    from deft_amd.attention import AttentionPlan
    from deft_amd.hiplib import DeftHipError
    g = torch.Generator().manual_seed(0)
    q, k, pos, qs = torch.randn(5, 2, 32, generator=g), torch.randn(5, 1, 32, generator=g), torch.arange(5, dtype=torch.int32).view(5, 1), torch.tensor([0, 5], dtype=torch.int32)
    a, b = (AttentionPlan(2, 1, 32, axes=(16,), device="cpu", lib=x) for x in (emu_lib, emu_lib.twin()))
    for x, y in zip(a.rotate(q, k, pos) + (a.attend(q, k, k, qs),), b.rotate(q, k, pos) + (b.attend(q, k, k, qs),)):
        assert torch.equal(x, y)
    p40 = AttentionPlan(2, 1, 40, device="cpu", lib=emu_lib.twin())
    with pytest.raises(DeftHipError, match="deft_attn_p3 failed.*D=40"):
        p40.attend(torch.zeros(5, 2, 40), torch.zeros(5, 1, 40), torch.zeros(5, 1, 40), qs)
    with pytest.raises(DeftHipError, match="deft_attn_ws_floats_p3 failed.*D=40"):
        p40.attend(torch.zeros(5, 2, 40), torch.zeros(5, 1, 40), torch.zeros(5, 1, 40), qs, max_k=500)
    so = build.build(force=False, verbose=False)
    names = subprocess.check_output(["nm", so], text=True).split()
    for kernel in ("rotary_kernel", "attn_prompt_kernel", "attn_step_kernel", "attn_merge_kernel"):
        stubs = [n for n in names if "__device_stub__" + kernel in n]
        assert stubs and len(stubs) == len(set(stubs)), kernel


def test_written_rows_share_no_elements(emu_lib):
    """Outputs and caches whose rows overlap in any way are refused; strides that only look so are taken."""
    from deft_amd.attention import AttentionPlan
    from deft_amd.hiplib import DeftHipError
    g = torch.Generator().manual_seed(0)
    plan = AttentionPlan(4, 2, 32, axes=(16,), device="cpu", lib=emu_lib)
    q, k, pos, qs = torch.randn(4, 4, 32, generator=g), torch.randn(4, 2, 32, generator=g), torch.arange(4, dtype=torch.int32).view(4, 1), torch.tensor([0, 4], dtype=torch.int32)
    row = torch.arange(4, dtype=torch.int32)
    S = lambda t, h, ld, hs: torch.zeros(4096).as_strided((t, h, 32), (ld, hs, 1))  # noqa: E731
    want, (wq, wk) = plan.attend(q, k, k, qs), plan.rotate(q, k, pos)
    for ld, hs in ((64, 32), (32, 64), (96, 64), (160, 80), (96, 80)):                    # token 1 head 0 on token 0 head 2, ...
        with pytest.raises(DeftHipError, match="strides"):
            plan.attend(q, k, k, qs, out=S(4, 4, ld, hs))
        with pytest.raises(DeftHipError, match="strides"):
            plan.rotate(q, k, pos, out=(S(4, 4, ld, hs), None))
    for ld, hs in ((128, 32), (32, 128), (136, 32), (288, 64), (64, 288), (32 * 7, 32 * 2), (32 * 2, 32 * 9), (160, 96)):
        assert torch.equal(plan.attend(q, k, k, qs, out=S(4, 4, ld, hs)), want), (ld, hs)
        assert torch.equal(plan.rotate(q, k, pos, out=(S(4, 4, ld, hs), None))[0], wq), (ld, hs)
    with pytest.raises(DeftHipError, match="strides"):
        plan.rotate(q, k, pos, cache=(S(8, 2, 32, 64), None), row=row)                      # row 2 of head 0 is row 0 of head 1
    assert torch.equal(plan.rotate(q, k, pos, cache=(S(8, 2, 96, 64), None), row=row)[1][:4], wk)
    assert torch.equal(plan.rotate(q, k, pos, cache=(S(8, 2, 96, 32), None), row=row)[1][:4], wk)


MASKED = [dict(nq=(9, 3), nk=(140, 3), max_k=100),                   # step kernel, four waves
          dict(nq=(9, 3), nk=(140, 3), max_k=700),                   # the same, keys split
          dict(nq=(9, 3), nk=(140, 3), max_k=40),                    # one wave over long keys
          dict(nq=(150, 4), nk=(150, 4), max_k=None, cache=None),    # prompt kernel ... (max_k None: the average is above two tiles)
          dict(nq=(150, 4), nk=(150, 4), max_k=1100, cache=None),    # ... keys split
          dict(nq=(200, 30), nk=(333, 30), max_k=333)]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("late", [0, 1])
def test_masked_values(emu_lib, dt, D, late):
    emu_lib.cdll.hipemu_set_late_dma(late)                           # (LDS fetches delivered when issued, or when waited for)
    try:
        for i, kw in enumerate(MASKED):
            ae.check_masked_values(emu_lib, "cpu", dt, D, (float("nan"), float("inf"), float("-inf"))[(i + late + D // 32) % 3], **kw)
    finally:
        emu_lib.cdll.hipemu_set_late_dma(0)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_seen_infinities(emu_lib, dt, D):
    for kw in MASKED:
        ae.check_seen_infinities(emu_lib, "cpu", dt, D, **kw)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_step_kernels_keep_whole_probabilities(emu_lib, dt, D):
    ae.check_two_piece_steps(emu_lib, "cpu", dt, D, (1, 1, 5), (60, 31, 5), None)             # one wave
    ae.check_two_piece_steps(emu_lib, "cpu", dt, D, (1, 2), (900, 255), None)                 # four, keys split
    ae.check_two_piece_steps(emu_lib, "cpu", dt, D, (1, 2), (300, 255), 200)                  # four


@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_attend_in_place(emu_lib, dt):
    ae.check_in_place(emu_lib, "cpu", dt)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_sequences_that_share_keys(emu_lib, dt):
    ae.check_shared_keys(emu_lib, "cpu", dt)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_many_sequences(emu_lib, dt):
    ae.check_many_sequences(emu_lib, "cpu", dt, 1500)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("max_k", [40, None, 1100])
def test_far_scores_beside_masked_values(emu_lib, dt, max_k):
    ae.check_far_scores_beside_masked_values(emu_lib, "cpu", dt, max_k)


@pytest.mark.parametrize("dt,D", [(F32, 8), (F32, 24), (F32, 40), (F32, 200), (F32, 256), (F16, 16), (BF16, 48), (BF16, 80), (F16, 112), (BF16, 144), (F16, 240)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotary_widths(emu_lib, dt, D, norm):
    """Every head width between the powers of two, more tokens than a wave holds, an odd count of heads."""
    import attention_checks as ac
    v = 4 if dt == F32 else 8
    axes = (D // 2 // v * v,) if D < 4 * v else (v, D // 2 // v * v - v)
    ac.check_rotary(emu_lib, "cpu", dt, T=37, H=5, Hk=5, D=D, axes=axes, norm=norm, adjacent=D % 32 != 0, cache="rows" if norm else None)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("known", [False, True])
def test_one_long_sequence_among_short_ones(emu_lib, dt, known):
    """Packed histories and one clip: by the average length (the default estimate) and by the longest one, on either kernel."""
    import attention_checks as ac
    n = [1, 3, 0, 2] * 10 + [260] + [1, 5] * 20
    ac.check_attend(emu_lib, "cpu", dt, n, n, 4, 2, 64, max_k=260 if known else None)
