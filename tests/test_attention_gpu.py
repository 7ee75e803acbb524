"""-m gpu: deft_amd.attention on a real MI355X against plain implementations in 64 bits (tests/attention_checks.py)."""
import math

import pytest
import torch

import attention_checks as ac
from deft_amd.attention import AttentionPlan

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("kw", [
    dict(T=100, H=8, Hk=8, D=32, axes=(4, 6, 6), frac=True),
    dict(T=333, H=4, Hk=2, D=96, axes=(8, 12, 12), adjacent=True),
    dict(T=200, H=16, Hk=4, D=64, axes=(8, 12, 12), norm=True, cache="slots"),
    dict(T=37, H=4, Hk=4, D=32, axes=(3, 13), cache="rows", adjacent=True),
    dict(T=1, H=40, Hk=8, D=128, axes=(16, 24, 24), norm=True, weights=False),
    dict(T=61, H=2, Hk=2, D=256, axes=(64, 32, 32), far=True, inverse=True),
    dict(T=5001, H=5, Hk=1, D=64, axes=(16, 16), norm=True, inplace=True),
    dict(T=33001, H=1, Hk=1, D=32, axes=(8, 8), norm=True, cache="rows"),      # several tokens a wave, an odd count of them
    dict(T=9001, H=3, Hk=1, D=64, axes=(16, 16), adjacent=True),
])
def test_rotary(gpu_lib, dt, kw):
    ac.check_rotary(gpu_lib, "cuda", dt, **kw)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("kw", [
    dict(nq=[1], nk=[1], H=1, Hk=1, D=32),
    dict(nq=[5, 0, 1, 33], nk=[5, 0, 1, 33], H=4, Hk=2, D=64),
    dict(nq=[300, 7, 129, 128], nk=[300, 7, 129, 128], H=6, Hk=2, D=128),
    dict(nq=[257], nk=[1030], H=4, Hk=4, D=96),
    dict(nq=[140, 60], nk=[140, 60], H=4, Hk=1, D=64, causal=False),
    dict(nq=[40, 6], nk=[20, 0], H=2, Hk=1, D=32),
    dict(nq=[1, 1, 1, 1], nk=[700, 1, 0, 64], H=10, Hk=2, D=64, cache="slots", poison=True),
    dict(nq=[1], nk=[5000], H=8, Hk=1, D=128, cache="slots", poison=True),
    dict(nq=[9, 70], nk=[1300, 90], H=3, Hk=1, D=32, cache="slots", poison=True),
    dict(nq=[60, 33], nk=[60, 33], H=2, Hk=1, D=96, gap=70, poison=True, head_major=True),
    dict(nq=[1] * 70, nk=list(range(70)), H=4, Hk=4, D=32, cache="slots", poison=True),
])
def test_attend(gpu_lib, dt, kw):
    ac.check_attend(gpu_lib, "cuda", dt, **kw)


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_every_kernel(gpu_lib, dt, D):
    """Prompt and step kernels of every width and type, one wave or four, keys split or whole, causal or not, lengths that end inside tiles."""
    ac.check_attend(gpu_lib, "cuda", dt, [260, 33], [260, 33], 4, 2, D)                               # prompt
    ac.check_attend(gpu_lib, "cuda", dt, [130], [1500], 2, 1, D)                                      # prompt, keys split
    ac.check_attend(gpu_lib, "cuda", dt, [150, 90], [333, 90], 2, 1, D, causal=False, cache="slots", poison=True)
    ac.check_attend(gpu_lib, "cuda", dt, [1, 1, 5], [60, 31, 5], 6, 2, D, cache="slots", poison=True)  # step, one wave
    ac.check_attend(gpu_lib, "cuda", dt, [1, 2], [900, 255], 5, 1, D, cache="slots", poison=True)     # step, four waves, keys split
    ac.check_attend(gpu_lib, "cuda", dt, [1, 2], [900, 255], 5, 1, D, cache="slots", poison=True, max_k=1)    # one wave over long keys


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_masked_keys_take_no_part(gpu_lib, dt, bad):
    """Infinities and NaN in keys and values behind a row's last visible key: prompt and step kernel, whole and split."""
    def spoil(b):
        n = 0
        for (k, v), q in zip(b["keys"], b["queries"]):
            m = k.shape[0]
            if "slot" not in b and m == q.shape[0]:
                k[-1], v[-1], v[-2, :, ::3] = bad, bad, bad
                b["k"][n:n + m], b["v"][n:n + m] = k.to("cuda"), v.to("cuda")
            n += m
    for nq in ([37, 5], [300, 4]):
        b = ac.make_batch(dt, nq, nq, 2, 1, 64, "cuda", seed=2)
        plan = AttentionPlan(2, 1, 64, device="cuda")
        spoil(b)
        for max_k in (None, 1000):
            o = plan.attend(b["q"], b["k"], b["v"], b["q_start"], max_k=max_k)
            for i, n in enumerate(nq):
                got = o[b["starts"][i]:b["starts"][i + 1]]
                want, _, A, mag = ac.ref_attend(b["queries"][i], *b["keys"][i], plan.scale, True)
                ac.assert_attended("early rows", got[:n - 2], want[:n - 2], A[:n - 2], mag[:n - 2], n, 64, dt)
                assert not torch.isfinite(got[n - 1]).all() and not torch.isfinite(got[n - 2, :, ::3]).any()


def layer(plan, x, wqkv, pos, q_start):
    """One attention layer over packed tokens, as a user runs it."""
    H, Hk, D = plan.heads, plan.kv_heads, plan.head_dim
    qkv = (x @ wqkv).view(x.shape[0], H + 2 * Hk, D)
    q, k = plan.norm_rotate(qkv[:, :H], qkv[:, H:H + Hk], pos)
    return plan.attend(q, k, qkv[:, H + Hk:], q_start)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_prompt_and_steps_agree(gpu_lib, dt):
    """The operators together: histories of 12 tracks in one packed prompt, against the same tokens fed one frame at a time through cache rows."""
    g = torch.Generator().manual_seed(0)
    B, cap, H, Hk, D = 12, 40, 8, 2, 64
    lens = [1 + (7 * i) % cap for i in range(B)]
    plan = AttentionPlan(H, Hk, D, axes=(8, 12, 12), q_weight=1 + 0.1 * torch.randn(D, generator=g), device="cuda")
    T = sum(lens)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    qkv = ac.rand(g, dt, T, H + 2 * Hk, D).cuda()
    pos = torch.stack([torch.arange(T), torch.randint(0, 600, (T,), generator=g), torch.randint(0, 1000, (T,), generator=g)], 1).to(torch.int32).cuda()
    q, k = plan.norm_rotate(qkv[:, :H], qkv[:, H:H + Hk], pos)
    whole = plan.attend(q, k, qkv[:, H + Hk:], torch.tensor(starts, dtype=torch.int32, device="cuda"))
    kc, vc = (torch.full((B + 1, cap, Hk, D), float("nan"), dtype=dt, device="cuda") for _ in range(2))
    steps = torch.empty_like(whole)
    for f in range(cap):
        live = [b for b in range(B) if lens[b] > f]
        if not live:
            break
        at = torch.tensor([starts[b] + f for b in live], device="cuda")
        slot = torch.tensor([B - b for b in live], dtype=torch.int32, device="cuda")
        x = qkv[at]
        qs, _ = plan.norm_rotate(x[:, :H], x[:, H:H + Hk], pos[at], v=x[:, H + Hk:], cache=(kc, vc), row=slot * cap + f)
        assert torch.equal(qs, q[at])
        q_start = torch.arange(len(live) + 1, dtype=torch.int32, device="cuda")
        steps[at] = plan.attend(qs, kc, vc, q_start, slot=slot, k_len=torch.full((len(live),), f + 1, dtype=torch.int32, device="cuda"))
    for b in range(B):
        s = slice(starts[b], starts[b + 1])
        want, _, A, mag = ac.ref_attend(q[s].cpu(), k[s].cpu(), qkv[s, H + Hk:].cpu(), plan.scale, True)
        ac.assert_attended("prompt %d" % b, whole[s], want, A, mag, lens[b], D, dt)
        ac.assert_attended("steps %d" % b, steps[s], want, A, mag, lens[b], D, dt)


def test_graph_replays(gpu_lib):
    """A captured layer and a captured split step: replayed with new inputs between eager work, each replay equal to the eager call."""
    g = torch.Generator(device="cuda").manual_seed(3)
    plan = AttentionPlan(8, 2, 64, axes=(8, 12, 12), device="cuda")
    x = torch.randn(150, 256, generator=g, device="cuda", dtype=BF16)
    w = torch.randn(256, 12 * 64, generator=g, device="cuda", dtype=BF16) / 16
    pos = torch.randint(0, 999, (150, 3), generator=g, device="cuda", dtype=torch.int32)
    qs = torch.tensor([0, 50, 150], dtype=torch.int32, device="cuda")
    q1, kc = torch.randn(2, 8, 64, generator=g, device="cuda", dtype=BF16), torch.randn(2, 9000, 2, 64, generator=g, device="cuda", dtype=BF16)
    i2, slot, ln = torch.arange(3, device="cuda", dtype=torch.int32), torch.tensor([1, 0], dtype=torch.int32, device="cuda"), torch.tensor([8999, 5], dtype=torch.int32, device="cuda")
    both = lambda: (layer(plan, x, w, pos, qs), plan.attend(q1, kc, kc, i2, slot=slot, k_len=ln))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = both()
        graphs.append((gr, got))
    for r in range(4):
        x.copy_(torch.randn(150, 256, generator=g, device="cuda"))
        q1.copy_(torch.randn(2, 8, 64, generator=g, device="cuda"))
        ln[0] = 8999 - 700 * r
        want = both()
        torch.cuda.synchronize()
        for gr, got in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_streams_and_repeats(gpu_lib):
    """The same split call on two streams at once, many times: the same bits every time."""
    g = torch.Generator(device="cuda").manual_seed(5)
    plan = AttentionPlan(16, 2, 128, device="cuda")
    ins = [(torch.randn(3, 16, 128, generator=g, device="cuda", dtype=BF16), torch.randn(3, 6000, 2, 128, generator=g, device="cuda", dtype=BF16)) for _ in range(2)]
    qs, slot = torch.arange(4, device="cuda", dtype=torch.int32), torch.arange(3, device="cuda", dtype=torch.int32)
    ln = torch.tensor([6000, 17, 3111], dtype=torch.int32, device="cuda")
    want = [plan.attend(q, k, k, qs, slot=slot, k_len=ln) for q, k in ins]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                q, k = ins[i]
                got.append((i, plan.attend(q, k, k, qs, slot=slot, k_len=ln)))
    torch.cuda.synchronize()
    for i, o in got:
        assert torch.equal(o, want[i])


def test_offsets_past_32_bits(gpu_lib):
    """A cache of more than 2^31 elements: the last slot's keys and a packed start far behind."""
    plan = AttentionPlan(2, 1, 128, device="cuda")
    S, cap = 3, 6_000_000                                            # 3 x 6e6 x 128 = 2.3e9 elements, 4.6 GB in fp16
    k = torch.zeros(S, cap, 1, 128, dtype=F16, device="cuda")
    m = 40
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(m, 1, 128, generator=g, device="cuda").half()
    q = torch.randn(1, 2, 128, generator=g, device="cuda").half()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k[2, :m] = rows
    o = plan.attend(q, k, k, i32(0, 1), slot=i32(2), k_len=i32(m), max_k=m)
    want, _, A, mag = ac.ref_attend(q.cpu(), rows.cpu(), rows.cpu(), plan.scale, True)
    ac.assert_attended("slot 2", o, want, A, mag, m, 128, F16)
    k[2, cap - m:] = rows
    flat = k.view(S * cap, 1, 128)
    o = plan.attend(q, flat, flat, i32(0, 1), k_start=i32(S * cap - m), k_len=i32(m), max_k=m)
    ac.assert_attended("last rows", o, want, A, mag, m, 128, F16)
    # the last row of the cache as a destination of norm_rotate
    p2 = AttentionPlan(2, 1, 128, axes=(64,), device="cuda")
    _, kc = p2.rotate(q, rows[:1], i32(0).view(1, 1), cache=(k, None), row=i32(S * cap - 1))
    assert torch.equal(k[2, cap - 1], rows[0])


def test_far_positions_keep_their_angle(gpu_lib):
    plan = AttentionPlan(1, 1, 64, axes=(32,), device="cuda")
    q = torch.ones(3, 1, 64, device="cuda")
    pos = torch.tensor([[2_000_000_000], [-2_000_000_000], [1]], dtype=torch.int32, device="cuda")
    got, _ = plan.rotate(q, None, pos)
    want, mag = ac.ref_rotate(q, pos, [10000.0 ** (-i / 32) for i in range(32)], [0] * 32, False)
    ac.assert_rotated("far", got, want, mag, F32)
