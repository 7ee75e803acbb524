"""-m gpu: corners of the attention-layer operators on a real MI355X; the checks themselves are in tests/attention_edges.py."""
import pytest
import torch

import attention_edges as ae

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_key_rows_that_share_memory(gpu_lib, dt, bad):
    ae.check_shared_key_rows(gpu_lib, "cuda", dt, bad)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_unturned_elements(gpu_lib, dt, adjacent, norm):
    ae.check_unturned_elements(gpu_lib, "cuda", dt, adjacent, norm)


@pytest.mark.parametrize("dt,size,eps", [(F32, 1e25, 1e-6), (BF16, 1e30, 1e-6), (F32, 3e37, 0.0), (F32, 1e-25, 0.0), (BF16, 1e-30, 0.0), (F32, 1e-20, 1e-38), (F16, 1e-5, 0.0),
                                         (F32, 1e-30, 1e-6), (BF16, 1e19, 1e-6)])
def test_norm_of_far_values(gpu_lib, dt, size, eps):
    ae.check_norm_of_far_values(gpu_lib, "cuda", dt, size, eps)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_norm_of_far_values_among_others(gpu_lib, dt):
    """Waves of several passes, a far head in the last: what the earlier passes have written in place is not read again."""
    ae.check_norm_of_far_values(gpu_lib, "cuda", dt, 1e25, 1e-6, T=1400, H=80 if dt == F32 else 160, D=32, R=16, inplace=True)


FAR = [dict(size=s, equal=e) for s in (1e8, -1e8, 1e12, -1e12, 1e30, -1e30, 2e38, -2e38, -3e38, 3e38) for e in (True, False) if e or abs(s) < 1e38]


@pytest.mark.parametrize("kw", FAR)
@pytest.mark.parametrize("dt", [F32, BF16])
def test_far_scores(gpu_lib, dt, kw):
    for D in (32, 64, 96, 128):
        ae.check_far_scores(gpu_lib, "cuda", dt, D=D, **kw)                                                    # one-wave step kernel
        ae.check_far_scores(gpu_lib, "cuda", dt, D=D, nq=(2, 3), nk=(300, 40), max_k=300, cache="slots", **kw)     # four waves
        ae.check_far_scores(gpu_lib, "cuda", dt, D=D, nq=(1,), nk=(600,), max_k=600, cache="slots", **kw)          # keys split
        ae.check_far_scores(gpu_lib, "cuda", dt, D=D, nq=(80,), nk=(90,), **kw)                                # prompt kernel
        ae.check_far_scores(gpu_lib, "cuda", dt, D=D, nq=(70,), nk=(600,), max_k=1100, causal=False, **kw)     # prompt, split


@pytest.mark.parametrize("size", [1e5, -1e5, 1e8, -1e8])
def test_far_scores_fp16(gpu_lib, size):
    for equal in (True, False):
        ae.check_far_scores(gpu_lib, "cuda", F16, size, equal=equal)
        ae.check_far_scores(gpu_lib, "cuda", F16, size, nq=(80,), nk=(90,), equal=equal)


def test_starts_that_do_not_grow(gpu_lib, monkeypatch):
    empty = torch.empty                                              # the workspace is NaN
    monkeypatch.setattr(torch, "empty", lambda *a, **k: empty(*a, **k).fill_(float("nan")) if k.get("dtype") is torch.float32 else empty(*a, **k))
    ae.check_starts_that_do_not_grow(gpu_lib, "cuda")


def test_plan_made_on_another_stream(gpu_lib):
    """A plan's copies of its weights are there when the plan is: made on a stream that is still busy producing them, used at once on another one."""
    from deft_amd.attention import AttentionPlan
    g = torch.Generator(device="cuda").manual_seed(0)
    q, pos = torch.randn(64, 4, 64, generator=g, device="cuda"), torch.arange(64, device="cuda", dtype=torch.int32).view(64, 1)
    w = torch.rand(64, generator=g, device="cuda") + 0.5
    want = AttentionPlan(4, 1, 64, axes=(32,), q_weight=w, device="cuda").norm_rotate(q, None, pos)[0]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(a):
            x = big
            for _ in range(20):
                x = (x @ big) * 1e-2                                  # some milliseconds of work in front of the weights
            late = w + 0.0 * x[0, :64].nan_to_num(0.0, 0.0, 0.0)
            plan = AttentionPlan(4, 1, 64, axes=(32,), q_weight=late, device="cuda")
        with torch.cuda.stream(b):
            got = plan.norm_rotate(q, None, pos)[0]
        b.synchronize()
        assert torch.equal(got, want)
        a.synchronize()


MASKED = [dict(nq=(9, 3), nk=(140, 3), max_k=100),                   # step kernel, four waves
          dict(nq=(9, 3), nk=(140, 3), max_k=700),                   # the same, keys split
          dict(nq=(9, 3), nk=(140, 3), max_k=40),                    # one wave over long keys
          dict(nq=(150, 4), nk=(150, 4), max_k=None, cache=None),    # prompt kernel ... (max_k None: the average is above two tiles)
          dict(nq=(150, 4), nk=(150, 4), max_k=1100, cache=None),    # ... keys split
          dict(nq=(200, 30), nk=(333, 30), max_k=333)]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_masked_values(gpu_lib, dt, D, bad):
    for kw in MASKED:
        ae.check_masked_values(gpu_lib, "cuda", dt, D, bad, **kw)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_seen_infinities(gpu_lib, dt, D):
    for kw in MASKED:
        ae.check_seen_infinities(gpu_lib, "cuda", dt, D, **kw)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_step_kernels_keep_whole_probabilities(gpu_lib, dt, D):
    ae.check_two_piece_steps(gpu_lib, "cuda", dt, D, (1, 1, 5), (60, 31, 5), None)             # one wave
    ae.check_two_piece_steps(gpu_lib, "cuda", dt, D, (1, 2), (900, 255), None)                 # four, keys split
    ae.check_two_piece_steps(gpu_lib, "cuda", dt, D, (1, 2), (300, 255), 200)                  # four


@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_attend_in_place(gpu_lib, dt):
    ae.check_in_place(gpu_lib, "cuda", dt)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_sequences_that_share_keys(gpu_lib, dt):
    ae.check_shared_keys(gpu_lib, "cuda", dt)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_many_sequences(gpu_lib, dt):
    ae.check_many_sequences(gpu_lib, "cuda", dt, 40000)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("max_k", [40, None, 1100])
def test_far_scores_beside_masked_values(gpu_lib, dt, max_k):
    ae.check_far_scores_beside_masked_values(gpu_lib, "cuda", dt, max_k)


@pytest.mark.parametrize("dt,D", [(F32, 8), (F32, 24), (F32, 40), (F32, 200), (F32, 256), (F16, 16), (BF16, 48), (BF16, 80), (F16, 112), (BF16, 144), (F16, 240)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotary_widths(gpu_lib, dt, D, norm):
    """Every head width between the powers of two, more tokens than a wave holds, an odd count of heads."""
    import attention_checks as ac
    v = 4 if dt == F32 else 8
    axes = (D // 2 // v * v,) if D < 4 * v else (v, D // 2 // v * v - v)
    ac.check_rotary(gpu_lib, "cuda", dt, T=37, H=5, Hk=5, D=D, axes=axes, norm=norm, adjacent=D % 32 != 0, cache="rows" if norm else None)


def test_graphs_that_share_a_pool(gpu_lib):
    """Two captured split calls whose workspaces come from one memory pool, replayed in turns with eager calls between them: the eager bits every time.  (In
    the order of their capture, as torch asks of graphs that share a pool: the second one's output may stand where the first one's workspace was.)"""
    from deft_amd.attention import AttentionPlan
    g = torch.Generator(device="cuda").manual_seed(5)
    plan = AttentionPlan(8, 2, 64, device="cuda")
    qs, slot = torch.arange(3, device="cuda", dtype=torch.int32), torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    ln = torch.tensor([5000, 900], dtype=torch.int32, device="cuda")
    ins = [(torch.randn(2, 8, 64, generator=g, device="cuda", dtype=BF16), torch.randn(2, 5000, 2, 64, generator=g, device="cuda", dtype=BF16)) for _ in range(2)]
    call = lambda i: plan.attend(ins[i][0], ins[i][1], ins[i][1], qs, slot=slot, k_len=ln)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(0), call(1)
    torch.cuda.current_stream().wait_stream(side)
    graphs, pool = [], None
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=pool):
            got = call(i)
        pool = gr.pool()
        graphs.append((gr, got))
    for r in range(4):
        for i in range(2):
            ins[i][0].copy_(torch.randn(2, 8, 64, generator=g, device="cuda"))
        want = [call(0), call(1)]
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(graphs[i][1], want[i])


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("known", [False, True])
def test_one_long_sequence_among_short_ones(gpu_lib, dt, known):
    """Packed histories and one clip: by the average length (the default estimate) and by the longest one, on either kernel."""
    import attention_checks as ac
    n = [1, 3, 0, 2] * 10 + [1500] + [1, 5] * 20
    ac.check_attend(gpu_lib, "cuda", dt, n, n, 4, 2, 64, max_k=1500 if known else None)
