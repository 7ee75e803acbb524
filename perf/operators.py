"""The attention-layer operators of deft_amd.attention and what they are measured on.

A token is one detection of one frame (or one cell of a feature map) with a position (frame, y, x): the same objects whose embeddings the affinity
estimator compares and whose histories the LSTM motion model follows.  Three operators make an attention layer over such tokens:

  rotate        rotary positions with several axes on queries and keys
  norm_rotate   RMS norm of every query and key head and the rotation in one pass, keys and values written to cache rows where there is a cache
  attend        causal attention with grouped heads over packed sequences of different lengths, whole prompts or single tokens over a cache

`run` computes them in plain torch operations, or (`own`) by the calls a user makes of the framework.
"""
import math
import random

import torch

own = False
EPS = 1e-6
THETA = 10000.0
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases -----------------------------------------------------------------------------------------------------------------------------

def _rot(op, dtype, tokens, heads, kv_heads, dim, axes, adjacent=False, frac=False, cache=False):
    return {"op": op, "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "axes": axes,
            "adjacent": adjacent, "frac": frac, "cache": cache}


def _att(dtype, seqs, q_min, q_max, past_min, past_max, heads, kv_heads, dim, causal=True):
    """Sequence b has q_min..q_max queries and past_min..past_max keys before them; past_max = 0: keys are the prompt itself, else rows of a cache."""
    return {"op": "attend", "dtype": dtype, "seqs": seqs, "q_min": q_min, "q_max": q_max, "past_min": past_min, "past_max": past_max,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "causal": causal}


def listed():
    return [
        # the detections of one frame (K = 100), sub-pixel centres as positions, the framework's own fp32: the smallest call, latency
        dict(_rot("rotate", "fp32", 100, 8, 8, 32, "4/6/6", frac=True), name="rotate frame"),
        # every cell of the stride-16 map of a 1088 x 608 clip of eight frames (38 x 68 each), adjacent pairs, a third of the head not rotated
        dict(_rot("rotate", "fp16", 20672, 12, 12, 96, "8/12/12", adjacent=True), name="rotate clip"),
        # one step of 200 live tracks: one token a track, keys and values into the cache rows of its history
        dict(_rot("norm_rotate", "bf16", 200, 16, 4, 64, "8/12/12", cache=True), name="norm step"),
        # the stored frames of a recorder (50 frames of 100 detections) in fp32
        dict(_rot("norm_rotate", "fp32", 5000, 8, 2, 128, "16/24/24", frac=True), name="norm stored frames"),
        # a packed prompt of long clips
        dict(_rot("norm_rotate", "bf16", 32781, 32, 8, 128, "16/24/24"), name="norm prompt"),
        # histories of 200 tracks, 1 to 50 observations each, packed
        dict(_att("bf16", 200, 1, 50, 0, 0, 16, 4, 64), name="track histories"),
        # 500 history objects in fp32
        dict(_att("fp32", 500, 1, 50, 0, 0, 8, 8, 32), name="track histories fp32"),
        # six clips of different lengths in one batch
        dict(_att("fp16", 6, 300, 5000, 0, 0, 16, 4, 64), name="ragged clips"),
        # one long sequence
        dict(_att("bf16", 1, 16384, 16384, 0, 0, 16, 4, 128), name="long clip"),
        # new frames of running streams: chunks of up to 300 tokens over the keys already there
        dict(_att("bf16", 8, 1, 300, 500, 5000, 12, 4, 96), name="chunks over a cache"),
        # one token for each of 200 tracks over its history
        dict(_att("bf16", 200, 1, 1, 0, 50, 16, 4, 64), name="track step"),
        # one token for each of 24 streams over long histories
        dict(_att("bf16", 24, 1, 1, 2000, 32000, 32, 8, 128), name="stream step"),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    dim = rng.choice([32, 64, 96, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5])
    kind = rng.choice(["rotate", "norm_rotate", "prompt", "chunk", "step"])
    if kind in ("rotate", "norm_rotate"):
        pairs = dim // 2 if rng.random() < 0.7 else dim // 2 - 8
        a = rng.randrange(1, pairs // 2)
        b = rng.randrange(1, pairs - a)
        axes = rng.choice(["%d/%d/%d" % (a, b, pairs - a - b), "%d/%d" % (a, pairs - a)])
        most = 32000 * 40 * 128 // ((heads + 2 * kv_heads) * dim * (2 if dtype == "fp32" else 1))
        return _rot(kind, dtype, _between(rng, 1, min(60000, most)), heads, kv_heads, dim, axes, adjacent=rng.random() < 0.5,
                    frac=rng.random() < 0.3, cache=kind == "norm_rotate" and rng.random() < 0.5)
    if kind == "prompt":
        seqs = _between(rng, 1, 300)
        q_max = _between(rng, 1, min(8000, 16000 // int(math.sqrt(seqs))))
        q_min = max(1, int(q_max * rng.choice([0.02, 0.3, 1.0])))
        while seqs * q_max * q_max * heads * (4 if dtype == "fp32" else 1) > 16384 * 16384 * 16:
            q_max = max(1, q_max * 2 // 3)
            q_min = min(q_min, q_max)
        return _att(dtype, seqs, q_min, q_max, 0, 0, heads, kv_heads, dim, causal=rng.random() < 0.8)
    seqs = _between(rng, 1, 256)
    q_max = 1 if kind == "step" else _between(rng, 2, 400)
    past_max = _between(rng, 2, 32000)
    while seqs * past_max * kv_heads * dim * (2 if dtype == "fp32" else 1) > 24 * 32000 * 8 * 128 or seqs * past_max * q_max * heads > 16384 * 16384 * 8:
        past_max = max(2, past_max * 2 // 3)
        seqs = max(1, seqs * 4 // 5)
    return _att(dtype, seqs, 1, q_max, max(0, int(past_max * rng.choice([0.0, 0.1, 0.9]))), past_max, heads, kv_heads, dim)


def _lengths(case):
    """(queries, keys) of every sequence of an `attend` case; the case alone decides them."""
    r = random.Random(case["seqs"] * 1000003 + case["q_max"] * 1009 + case["past_max"])
    nq = [r.randint(case["q_min"], case["q_max"]) for _ in range(case["seqs"])]
    nk = [n + (r.randint(case["past_min"], case["past_max"]) if case["past_max"] else 0) for n in nq]
    return nq, nk


# ---- inputs --------------------------------------------------------------------------------------------------------------------------------

def _rand(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, H, Hk, D = TYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "attend":
        nq, nk = _lengths(case)
        Tq, B = sum(nq), case["seqs"]
        s = {"case": case, "nq": nq, "nk": nk, "scale": 1.0 / math.sqrt(D)}
        starts = [0]
        for n in nq:
            starts.append(starts[-1] + n)
        s["q_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        if case["past_max"]:
            cap = max(nk) + 3                       # rows of a slot; what stands behind a sequence's last key is old memory
            s["q"] = _rand(g, dt, Tq, H, D)
            s["k"], s["v"] = _rand(g, dt, B + 2, cap, Hk, D), _rand(g, dt, B + 2, cap, Hk, D)
            s["slot"] = torch.randperm(B + 2, generator=g, device="cuda")[:B].to(torch.int32)
            s["k_len"] = torch.tensor(nk, dtype=torch.int32, device="cuda")
        else:                                       # queries, keys and values as one projection leaves them
            qkv = _rand(g, dt, Tq, H + 2 * Hk, D)
            s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        if own:
            from deft_amd.attention import AttentionPlan
            s["plan"] = AttentionPlan(H, Hk, D)
        return s
    T = case["tokens"]
    axes = [int(a) for a in case["axes"].split("/")]
    R, norm = sum(axes), case["op"] == "norm_rotate"
    qkv = _rand(g, dt, T, H + 2 * Hk, D)
    s = {"case": case, "q": qkv[:, :H], "k": qkv[:, H:H + Hk], "v": qkv[:, H + Hk:]}
    span = torch.tensor([4000.0, 608.0, 1088.0], device="cuda")[:len(axes)]
    pos = torch.rand(T, len(axes), generator=g, device="cuda") * span
    s["pos"] = pos.contiguous() if case["frac"] else pos.to(torch.int32)
    s["freq"] = torch.tensor([THETA ** (-i / R) for i in range(R)], dtype=torch.float64, device="cuda")
    s["axis"] = torch.tensor([a for a, n in enumerate(axes) for _ in range(n)], device="cuda")
    if norm:
        s["qw"], s["kw"] = (1.0 + 0.2 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    if case["cache"]:
        rows = 2 * T + 5
        s["kc"], s["vc"] = _rand(g, dt, rows, Hk, D), _rand(g, dt, rows, Hk, D)
        s["row"] = torch.randperm(rows, generator=g, device="cuda")[:T].to(torch.int32)
    if own:
        from deft_amd.attention import AttentionPlan
        s["plan"] = AttentionPlan(H, Hk, D, axes=axes, theta=THETA, adjacent=case["adjacent"], eps=EPS,
                                  q_weight=s["qw"] if norm else None, k_weight=s["kw"] if norm else None)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------------------------

def run(s):
    op, cache = s["case"]["op"], s["case"].get("cache")
    if own:
        plan = s["plan"]
        if op == "rotate":
            return plan.rotate(s["q"], s["k"], s["pos"])
        if op == "norm_rotate":
            if not cache:
                return plan.norm_rotate(s["q"], s["k"], s["pos"])
            return plan.norm_rotate(s["q"], s["k"], s["pos"], v=s["v"], cache=(s["kc"], s["vc"]), row=s["row"])[0], s["kc"], s["vc"]
        if s["case"]["past_max"]:
            return plan.attend(s["q"], s["k"], s["v"], s["q_start"], slot=s["slot"], k_len=s["k_len"])
        return plan.attend(s["q"], s["k"], s["v"], s["q_start"], causal=s["case"]["causal"])
    if op == "attend":
        return _plain_attend(s)
    angle = s["pos"][:, s["axis"]].double() * s["freq"]             # (64 bits: at far positions a 32-bit product loses the angle)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _plain_rotate(s["q"], cos, sin, s["case"]["adjacent"], s.get("qw"))
    k = _plain_rotate(s["k"], cos, sin, s["case"]["adjacent"], s.get("kw"))
    if not cache:
        return q, k
    row = s["row"].long()
    s["kc"][row] = k
    s["vc"][row] = s["v"]
    return q, s["kc"], s["vc"]


def _plain_rotate(x, cos, sin, adjacent, weight):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight
    R = cos.shape[-1]
    if adjacent:
        a, b = y[..., 0:2 * R:2], y[..., 1:2 * R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :R], y[..., R:2 * R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., 2 * R:]), -1).to(x.dtype)


def _plain_attend(s):
    """Every sequence padded to the longest, one batched product for the scores and one for the values."""
    q, case = s["q"], s["case"]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    B, Lq, Lk, dev = case["seqs"], max(s["nq"]), max(s["nk"]), q.device
    start = s["q_start"].long()
    nq = start[1:] - start[:-1]
    nk = s["k_len"].long() if case["past_max"] else nq
    i, j = torch.arange(Lq, device=dev), torch.arange(Lk, device=dev)
    at_q = (start[:-1, None] + i).clamp(max=q.shape[0] - 1)                                      # [B, Lq]
    there = j < nk[:, None]                                                                      # [B, Lk]
    if case["past_max"]:
        at = torch.where(there, j, 0)
        k, v = (x[s["slot"].long()[:, None], at].float() for x in (s["k"], s["v"]))              # [B, Lk, Hk, D]
    else:
        at = torch.where(there, start[:-1, None] + j, 0)
        k, v = (x[at].float() for x in (s["k"], s["v"]))
    G = H // Hk
    qs = (q[at_q].float() * s["scale"]).view(B, Lq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Lq, D)
    p = torch.matmul(qs, k.permute(0, 2, 3, 1)).view(B, Hk, G, Lq, Lk)
    seen = there[:, None, :]                                                                     # [B, 1 or Lq, Lk]
    if case["causal"]:
        seen = seen & (j <= (nk - nq)[:, None, None] + i[:, None])
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p -= p.amax(-1, keepdim=True).clamp(min=-3e38)
    p.exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hk, G * Lq, Lk), v.permute(0, 2, 1, 3)).view(B, Hk, G, Lq, D)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Lq, H, D)[i < nq[:, None]].to(q.dtype)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    turn = torch.zeros(case["tokens"], case["dim"] // 2, dtype=torch.float64, device="cuda")
    R = s["freq"].numel()
    turn[:, :R] = s["pos"].double().gather(1, s["axis"].expand(case["tokens"], R)) * s["freq"]
    turn = torch.polar(torch.ones_like(turn[:, :R]), turn[:, :R])[:, None]
    got = []
    for x, w in ((s["q"], s.get("qw")), (s["k"], s.get("kw"))):
        y = x.double()
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt() * w.double()
        z = torch.complex(y[..., 0:2 * R:2], y[..., 1:2 * R:2]) if case["adjacent"] else torch.complex(y[..., :R].contiguous(), y[..., R:2 * R].contiguous())
        z = z * turn
        if case["adjacent"]:
            y[..., 0:2 * R:2], y[..., 1:2 * R:2] = z.real, z.imag
        else:
            y[..., :R], y[..., R:2 * R] = z.real, z.imag
        got.append(y)
    if not case["cache"]:
        return got[0], got[1]
    kc, vc, row = s["kc"].double(), s["vc"].double(), s["row"].long()
    kc[row], vc[row] = got[1], s["v"].double()
    return got[0], kc, vc


def _exact_attend(s):
    case, G = s["case"], s["case"]["heads"] // s["case"]["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    t0 = 0
    for b, (n, m) in enumerate(zip(s["nq"], s["nk"])):
        if case["past_max"]:
            slot = int(s["slot"][b])
            k, v = s["k"][slot, :m], s["v"][slot, :m]
        else:
            k, v = s["k"][t0:t0 + n], s["v"][t0:t0 + n]
        late = None
        if case["causal"]:
            late = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        step = max(1, (1 << 28) // (n * m))         # query heads at a time
        for h in range(0, case["heads"], step):
            hs = torch.arange(h, min(h + step, case["heads"]), device="cuda")
            a = torch.einsum("nhd,mhd->hnm", s["q"][t0:t0 + n, hs].double(), k[:, hs // G].double()) * s["scale"]
            if late is not None:
                a.masked_fill_(late, -math.inf)
            out[t0:t0 + n, hs] = torch.einsum("hnm,mhd->nhd", torch.softmax(a, -1), v[:, hs // G].double())
        t0 += n
    return out


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------------

def work(case):
    size, H, Hk, D = TYPES[case["dtype"]].itemsize, case["heads"], case["kv_heads"], case["dim"]
    if case["op"] != "attend":
        n = case["tokens"] * D * (H + Hk)
        values = case["tokens"] * D * Hk if case["cache"] else 0
        return {"bytes": 2 * size * (n + values) + case["tokens"] * 4 * (len(case["axes"].split("/")) + bool(case["cache"])),
                "flops": (7 if case["op"] == "norm_rotate" else 3) * n}
    nq, nk = _lengths(case)
    pairs = sum(n * m - (n * (n - 1) // 2 if case["causal"] else 0) for n, m in zip(nq, nk))
    return {"bytes": size * D * (2 * H * sum(nq) + 2 * Hk * sum(nk)), "flops": 4 * D * H * pairs}
