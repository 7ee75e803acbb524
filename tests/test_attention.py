"""-m "not gpu": the attention-layer kernels through the SIMT emulator, and the refusals of deft_amd.attention."""
import pytest
import torch

import attention_checks as ac
from deft_amd.attention import AttentionPlan
from deft_amd.hiplib import DeftHipError

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("kw", [
    dict(T=5, H=8, Hk=8, D=32, axes=(4, 6, 6), frac=True),
    dict(T=3, H=4, Hk=2, D=96, axes=(8, 12, 12), adjacent=True),
    dict(T=7, H=3, Hk=1, D=64, axes=(8, 12, 12), norm=True),
    dict(T=9, H=4, Hk=2, D=64, axes=(24,), norm=True, cache="slots", adjacent=True),
    dict(T=6, H=4, Hk=4, D=32, axes=(3, 13), cache="rows"),
    dict(T=1, H=20, Hk=4, D=128, axes=(16, 24, 24), norm=True, weights=False),
    dict(T=4, H=2, Hk=2, D=256, axes=(64, 32, 32), far=True, inverse=True),
    dict(T=5, H=5, Hk=1, D=64, axes=(16, 16), inplace=True),
    dict(T=5, H=5, Hk=1, D=64, axes=(16, 16), norm=True, inplace=True, adjacent=True),
    dict(T=2, H=6, Hk=1, D=64, axes=(8,), k_none=True),
    dict(T=8201, H=1, Hk=1, D=32, axes=(8, 8), norm=True),                    # several tokens a wave, an odd count of them
    dict(T=16390, H=1, Hk=1, D=32, axes=(4, 4), adjacent=True, cache="rows"),
    dict(T=8195, H=2, Hk=1, D=96, axes=(24, 16), k_none=True),
])
def test_rotary(emu_lib, dt, kw):
    ac.check_rotary(emu_lib, "cpu", dt, **kw)


def test_rotate_and_back(emu_lib):
    g = torch.Generator().manual_seed(4)
    q, k = ac.rand(g, F32, 6, 4, 64), ac.rand(g, F32, 6, 2, 64)
    pos = torch.randint(-500, 500, (6, 3), generator=g, dtype=torch.int32)
    plan = AttentionPlan(4, 2, 64, axes=(8, 12, 12), device="cpu", lib=emu_lib)
    q1, k1 = plan.rotate(q, k, pos)
    q2, k2 = plan.rotate(q1, k1, pos, inverse=True)
    for a, b in ((q, q2), (k, k2)):
        a2 = a.abs()
        mag = a2 + a2.roll(32, -1)
        assert ((a - b).abs() <= 2 * 24 * ac.U * 2 * mag + 2 * ac.U * a2).all()


SHAPES = [
    dict(nq=[1], nk=[1], H=1, Hk=1, D=32),
    dict(nq=[5, 0, 1, 33], nk=[5, 0, 1, 33], H=4, Hk=2, D=64),
    dict(nq=[3, 2], nk=[70, 2], H=4, Hk=1, D=128),
    dict(nq=[40, 7], nk=[40, 7], H=2, Hk=2, D=96, causal=False),
    dict(nq=[4, 6], nk=[2, 0], H=2, Hk=1, D=32),                              # more queries than keys: rows that see nothing
    dict(nq=[1, 1, 1], nk=[66, 1, 0], H=6, Hk=2, D=64, cache="slots", poison=True),
    dict(nq=[9, 1], nk=[130, 5], H=3, Hk=1, D=32, cache="slots", poison=True),
    dict(nq=[6, 3], nk=[6, 3], H=2, Hk=1, D=64, gap=5, poison=True, head_major=True),
    dict(nq=[150], nk=[190], H=1, Hk=1, D=64),                                 # several tiles of keys and of rows
    dict(nq=[1, 2], nk=[600, 300], H=2, Hk=1, D=32, cache="slots", poison=True),   # split keys, joined
    dict(nq=[70], nk=[1100], H=1, Hk=1, D=32),                                 # the same for a prompt
    dict(nq=[1], nk=[520], H=5, Hk=1, D=128, cache="slots"),
]


@pytest.fixture(params=["early", "late"])
def dma(emu_lib, request):
    """LDS-DMA pieces delivered when they are issued, or only when their wave waits for them."""
    emu_lib.cdll.hipemu_set_late_dma(int(request.param == "late"))
    yield emu_lib
    emu_lib.cdll.hipemu_set_late_dma(0)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("kw", SHAPES)
def test_attend(dma, dt, kw):
    ac.check_attend(dma, "cpu", dt, **kw)


def _poison_last_keys(bad):
    def f(b):
        """The last two keys of every sequence hold `bad` values: only the last two queries may notice."""
        n = 0
        for (k, v), q in zip(b["keys"], b["queries"]):
            k[-1], v[-1], v[-2, :, ::3] = bad, bad, bad
            m = k.shape[0]
            b["k"][n:n + m], b["v"][n:n + m] = k.to(b["k"].device), v.to(b["v"].device)
            n += m
    return f


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_masked_keys_take_no_part(emu_lib, dt, bad):
    o = None
    b = ac.make_batch(dt, [37, 5], [37, 5], 2, 1, 64, "cpu", seed=2)
    plan = AttentionPlan(2, 1, 64, device="cpu", lib=emu_lib)
    clean = plan.attend(b["q"], b["k"], b["v"], b["q_start"])
    _poison_last_keys(bad)(b)
    o = plan.attend(b["q"], b["k"], b["v"], b["q_start"])
    early = torch.tensor([i for i in range(42) if i not in (35, 36, 40, 41)])
    assert torch.equal(o[early], clean[early])                                # every query before them: the same bits
    assert not torch.isfinite(o[36]).all() and not torch.isfinite(o[41]).all()
    assert not torch.isfinite(o[35, :, ::3]).any()                            # the key before the last: visible to query 35, where it is bad
    ok = [d for d in range(64) if d % 3]
    assert torch.equal(o[35][:, ok], clean[35][:, ok])


def test_starts_and_lengths_are_clamped(emu_lib):
    """Device-side values outside the tensors are cut to them, not read past them."""
    g = torch.Generator().manual_seed(1)
    q, k, v = ac.rand(g, F32, 4, 2, 32), ac.rand(g, F32, 3, 5, 1, 32), ac.rand(g, F32, 3, 5, 1, 32)
    plan = AttentionPlan(2, 1, 32, device="cpu", lib=emu_lib)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    o = plan.attend(q, k, v, i32(0, 1, 2, 3, 4), slot=i32(0, 7, -1, 2), k_len=i32(99, 5, 5, -3))
    want = plan.attend(q[:1], k, v, i32(0, 1), slot=i32(0), k_len=i32(5))
    assert torch.equal(o[:1], want) and (o[1:] == 0).all()
    kp = k.reshape(15, 1, 32)
    o = plan.attend(q, kp, kp, i32(0, 2, 99), k_start=i32(13, 40), k_len=i32(50, 3))
    want = plan.attend(q[:2], kp, kp, i32(0, 2), k_start=i32(13), k_len=i32(2))
    assert torch.equal(o[:2], want) and (o[2:] == 0).all()
    for bad in (i32(0, 4, 2, 4), i32(3, 1, 0, 4), i32(-7, 2, 99, 3), i32(4, 0, 4, 0)):      # starts that do not grow: some rows, but rows of q
        o = plan.attend(q, kp, kp, bad, out=torch.full((4, 2, 32), 5.0))
        assert torch.isfinite(o).all()
        o = plan.attend(q, kp, kp, bad, k_start=i32(0, 9, 14), k_len=i32(15, 15, 15), max_k=700, out=torch.full((4, 2, 32), 5.0))
    assert (plan.attend(q, kp[:0], kp[:0], i32(0, 4)) == 0).all()              # no keys at all
    assert plan.attend(q[:0], kp, kp, i32(0)).shape == (0, 2, 32)


def test_refusals(emu_lib):
    P = lambda **kw: AttentionPlan(**{**dict(heads=4, kv_heads=2, head_dim=64, axes=(8, 12, 12), device="cpu", lib=emu_lib), **kw})  # noqa: E731
    for kw, word in [(dict(heads=5), "multiple of kv_heads"), (dict(axes=(20, 20)), "pairs in all"), (dict(axis_of_pair=[3] * 32), "axis_of_pair"),
                     (dict(freq=[1.0]), "freq"), (dict(q_weight=torch.ones(3)), "q_weight")]:
        with pytest.raises(DeftHipError, match=word):
            P(**kw)
    plan = P()
    q, k, pos = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(3, 3, dtype=torch.int32)
    kc, row = torch.zeros(9, 2, 64), torch.zeros(3, dtype=torch.int32)
    for args, kw, word in [
            ((q.double(), k, pos), {}, "q is torch.float64"), ((q[:, :3], k, pos), {}, "q has shape"), ((q, k.half(), pos), {}, "k is torch.float16"),
            ((q, k[:2], pos), {}, "2 tokens"), ((q, k, pos[:, :2]), {}, "pos"), ((q, k, pos.long()), {}, "pos"), ((q, k, pos), {"v": k}, "v needs a cache"),
            ((q, k, pos), {"cache": (kc, None)}, "come together"), ((q, k, pos), {"cache": (kc, kc), "row": row}, "v and v_cache"),
            ((q, k, pos), {"cache": (kc, kc[:5]), "row": row, "v": k}, "rows"), ((q, k, pos), {"cache": (kc, None), "row": row.long()}, "row"),
            ((q, None, pos), {"cache": (kc, None), "row": row}, "need k"), ((q, k, pos), {"cache": (kc[:0], None), "row": row}, "empty"),
            ((torch.zeros(3, 4, 128)[..., ::2], k, pos), {}, "contiguous"), ((torch.zeros(3, 4, 66)[..., :64], k, pos), {}, "strides"),
            ((torch.zeros(769)[1:].view(3, 4, 64), k, pos), {}, "aligned"),
            ((q, k, pos), {"out": (torch.zeros(1, 4, 64).expand(3, 4, 64), None)}, "strides")]:
        with pytest.raises(DeftHipError, match=word):
            plan.rotate(*args, **kw)
    with pytest.raises(DeftHipError, match="without axes"):
        AttentionPlan(4, 2, 64, device="cpu", lib=emu_lib).rotate(q, k, pos)
    with pytest.raises(DeftHipError, match="R=13 pairs"):
        P(axes=(13,)).rotate(q.bfloat16(), k.bfloat16(), pos[:, :1].contiguous())
    with pytest.raises(DeftHipError, match="D=40"):
        AttentionPlan(4, 2, 40, device="cpu", lib=emu_lib).attend(torch.zeros(3, 4, 40), torch.zeros(3, 2, 40), torch.zeros(3, 2, 40), row[:2])
    cache, s2 = torch.zeros(2, 8, 2, 64), torch.zeros(1, dtype=torch.int32)
    qs = torch.tensor([0, 3], dtype=torch.int32)
    for args, kw, word in [
            ((q, k, k[:2], qs), {}, "k has shape"), ((q, k, k, qs.long()), {}, "q_start"), ((q, k, k, qs), {"slot": s2}, "slot needs a cache"),
            ((q, cache, cache, qs), {}, "needs slot and k_len"), ((q, cache, cache, qs), {"slot": s2, "k_len": qs}, "k_len"),
            ((q, k, k, qs), {"k_start": qs}, "k_start"), ((q, k.half(), k, qs), {}, "k is torch.float16"), ((q, k, k, qs), {"out": q[:2]}, "tokens")]:
        with pytest.raises(DeftHipError, match=word):
            plan.attend(*args, **kw)


def test_estimates_steer_only_the_split(dma):
    """max_k wrong in either direction, every kernel: one wave or four, prompt or step, keys split or not."""
    for dt in (F32, BF16):
        for max_k in (1, 700, 2 ** 40):
            ac.check_attend(dma, "cpu", dt, [1, 3], [330, 40], 2, 1, 64, cache="slots", poison=True, max_k=max_k)
            ac.check_attend(dma, "cpu", dt, [80], [600], 1, 1, 32, max_k=max_k)
            ac.check_attend(dma, "cpu", dt, [2, 40], [300, 40], 2, 2, 32, causal=False, cache="slots", max_k=max_k)


def test_gradients_are_refused(emu_lib):
    plan = AttentionPlan(2, 1, 32, axes=(16,), device="cpu", lib=emu_lib)
    q, k, pos, qs = torch.ones(2, 2, 32, requires_grad=True), torch.ones(2, 1, 32), torch.zeros(2, 1, dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32)
    for call in (lambda: plan.rotate(q, k, pos), lambda: plan.attend(q, k, k, qs), lambda: plan.attend(q.detach(), k, k.clone().requires_grad_(), qs)):
        with pytest.raises(DeftHipError, match="forward only"):
            call()
    with torch.no_grad():
        assert plan.attend(q, k, k, qs).shape == (2, 2, 32) and plan.rotate(q, k, pos)[0].shape == (2, 2, 32)


def test_many_heads_and_sequences(emu_lib):
    """More sequences than one lookup step takes, groups wider than a tile, gaps between nothing and nothing."""
    ac.check_attend(emu_lib, "cpu", F32, [1, 0, 2] * 170, [3, 1, 2] * 170, 1, 1, 32)
    ac.check_attend(emu_lib, "cpu", BF16, [3], [20], 150, 1, 32)
    ac.check_attend(emu_lib, "cpu", BF16, [2, 3], [90, 3], 135, 3, 32, cache="slots")


def test_descriptor_layouts_match_the_header():
    """ctypes mirrors of DeftRotary / DeftAttn: the header's fields in the header's order."""
    import os
    import re
    from deft_amd import hiplib
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "deft_hip.h")).read()
    for struct, mirror in (("DeftRotary", hiplib.RotaryDesc), ("DeftAttn", hiplib.AttnDesc)):
        body = src[src.index("typedef struct %s {" % struct):src.index("} %s;" % struct)]
        body = re.sub(r"/\*.*?\*/", "", body[body.index("{") + 1:], flags=re.S)
        names = []
        for decl in re.findall(r"(?:const void|const double|const int|const float|void|float|long long|int)\s*([^;]+);", body):
            names += [n.strip().lstrip("* ") for n in decl.split(",")]
        assert names == [n for n, _ in mirror._fields_]


def test_packed_descriptors_match_the_mirrors():
    """The struct formats that deft_amd.attention packs are the ctypes layouts: same size, same place for every field."""
    from deft_amd import attention, hiplib
    for fmt, mirror in ((attention._ROTARY, hiplib.RotaryDesc), (attention._ATTN, hiplib.AttnDesc)):
        vals = [i + 1 for i in range(len(mirror._fields_) - 1)] + [0.5]
        d = mirror.from_buffer_copy(fmt.pack(*vals))
        assert [getattr(d, n) for n, _ in mirror._fields_] == vals


def test_lds_fetches_keep_their_wait_states(tmp_path):
    """csrc/attn.hip writes its LDS-DMA out in assembly, where the compiler inserts no wait states: a scalar register that a vector instruction has written
    may be a memory instruction's source only five states later, and m0 one state after its write.  Checked on every one of the built code."""
    import os
    import re
    import subprocess
    from deft_amd import build
    build.build(force=False, verbose=False)
    llvm = "/opt/rocm/lib/llvm/bin/"
    if not os.path.exists(llvm + "llvm-objdump"):
        pytest.skip("llvm-objdump not in this image")
    fat, co = str(tmp_path / "fat.bin"), str(tmp_path / "dev.co")
    subprocess.check_call([llvm + "llvm-objcopy", "-O", "binary", "--only-section=.hip_fatbin", os.path.join(build.OBJ_DIR, "attn.hip.o"), fat])
    subprocess.check_call([llvm + "clang-offload-bundler", "--unbundle", "--type=o", "--input=" + fat, "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--output=" + co])
    code = [ln.split("//")[0].strip() for ln in subprocess.run([llvm + "llvm-objdump", "-d", co], capture_output=True, text=True).stdout.splitlines()]
    fetches = 0
    for i, ins in enumerate(code):
        m = re.match(r"buffer_load_dwordx4 v\d+, s\[(\d+):(\d+)\].* lds", ins)
        if not m:
            continue
        fetches += 1
        assert code[i - 1].startswith("s_nop") and code[i - 2].startswith("s_mov_b32 m0"), code[i - 3:i + 1]
        source, states, j = range(int(m[1]), int(m[2]) + 1), 0, i - 1
        while states < 5:
            w = re.match(r"v_read(?:first)?lane_b32 s(\d+)", code[j])
            assert not w or int(w[1]) not in source, code[j:i + 1]
            states += 1 + int(code[j].split()[1]) if code[j].startswith("s_nop") else 1
            j -= 1
    assert fetches > 100
