"""Speed and precision cases of the framework's attention-training operators: rotary positions with several axes, differential
attention, and AdamW over many tensors.

``run`` computes an operator in plain torch operations (``own`` false) or through the framework's entry points (``own`` true) on the
same inputs; ``exact`` gives the operator's values in 64 bits, from its definition.

    rotary   pair j of a head's first 2 P columns turns by pos[axis(j)] * theta^(-e(j)); P is split over the axes by `sections`
    diff     o = softmax(c q1 k1^T) v - lam_h softmax(c q2 k2^T) v, with q1, q2 (k1, k2) the head pair 2h, 2h + 1 and v twice as wide
    adamw    decoupled weight decay, moments in 32 bits or in 8 (blocks of 256 elements: m = s (c/127)|c/127|, sqrt(v) = s (c/255)^2)
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"
LR, B1, B2, EPS, WD, STEP0 = 1e-4, 0.9, 0.999, 1e-8, 0.1, 100
BLOCK = 256


def listed():
    rot = {"op": "rotary", "theta": 10000.0}
    diff = {"op": "diff"}
    adamw = {"op": "adamw"}
    return [
        # a new token of each of 8 sequences, far into its sequence, q and k of 12 heads: latency
        dict(rot, name="rotary one token", B=8, N=1, H=12, Hkv=12, dh=64, s0=8, s1=12, s2=12, ladder="shared", interleaved=False,
             far=True, dtype="bf16", train=False),
        # 16 volumes of 16 x 16 x 16 tokens and a class token in front of attention, 12 heads of 64 as the encoders have them; training
        dict(rot, name="rotary volumes", B=16, N=4097, H=12, Hkv=12, dh=64, s0=8, s1=12, s2=12, ladder="per_axis", interleaved=False,
             far=False, dtype="bf16", train=True),
        # slices of uneven length with shared key heads, part of a head's columns, neighbouring pairs, 32 bits
        dict(rot, name="rotary odd f32", B=3, N=1565, H=10, Hkv=2, dh=80, s0=8, s1=13, s2=15, ladder="shared", interleaved=True,
             far=True, dtype="f32", train=False),
        # two 256^3 volumes through an attention layer of width 768 (6 pairs of heads of 64): forward and gradients
        dict(diff, name="diff volumes train", B=2, Nq=4097, Nk=4097, H=6, Hkv=6, d=64, causal=False, lens=False, dtype="bf16", train=True),
        # short sequences of uneven length with shared key heads of 32, one of them empty: forward and gradients
        dict(diff, name="diff ragged train", B=6, Nq=333, Nk=333, H=8, Hkv=2, d=32, causal=True, lens=True, dtype="f16", train=True),
        # a long sequence read at once, causal, four query heads to a key head
        dict(diff, name="diff long causal", B=1, Nq=8192, Nk=8192, H=16, Hkv=4, d=64, causal=True, lens=False, dtype="bf16", train=False),
        # one token of each of 16 sequences against caches filled to different lengths
        dict(diff, name="diff one token", B=16, Nq=1, Nk=16384, H=16, Hkv=4, d=64, causal=True, lens=True, dtype="bf16", train=False),
        # a few tokens of one sequence against a cache, wide heads
        dict(diff, name="diff few tokens", B=1, Nq=7, Nk=5001, H=8, Hkv=2, d=128, causal=True, lens=False, dtype="f16", train=False),
        # the parameters of a 12-layer tower of width 640, all in 32 bits
        dict(adamw, name="adamw tower 32", width=640, layers=12, bits=32, dtype="f32"),
        # a tower of width 1024, 8-bit moments
        dict(adamw, name="adamw tower 8", width=1024, layers=8, bits=8, dtype="f32"),
        # a small 16-bit model, 8-bit moments: latency
        dict(adamw, name="adamw small 8", width=192, layers=2, bits=8, dtype="bf16"),
        # a small head in 16 bits, 32-bit moments: latency
        dict(adamw, name="adamw small 32", width=96, layers=1, bits=32, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "diff", "diff", "diff", "adamw"])
    if op == "rotary":
        dh = rng.choice([32, 64, 80, 96, 128])
        half = dh // 2 if rng.random() < 0.6 else dh // 2 - rng.randint(1, 7)
        s0, s1 = max(1, half // 4), max(1, (half - half // 4) // 2)
        Hkv = rng.choice([1, 2, 4, 8])
        H = Hkv * rng.choice([1, 2, 3])
        N = _log(rng, 1, 9000)
        B = _log(rng, 1, max(1, min(16, 100_000_000 // (N * (H + Hkv) * dh))))
        return {"op": op, "theta": rng.choice([10000.0, 500000.0]), "B": B, "N": N, "H": H, "Hkv": Hkv, "dh": dh, "s0": s0, "s1": s1,
                "s2": half - s0 - s1, "ladder": rng.choice(["shared", "per_axis"]), "interleaved": rng.random() < 0.3,
                "far": rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "train": rng.random() < 0.5}
    if op == "diff":
        kind = rng.choice(["train", "train", "read", "cache"])
        d = rng.choice([32, 64, 64, 128])
        Hkv = rng.choice([1, 2, 4])
        H = Hkv * rng.choice([1, 2, 4])
        dtype = rng.choice(["bf16", "bf16", "f16"])
        case = {"op": op, "H": H, "Hkv": Hkv, "d": d, "dtype": dtype, "train": kind == "train"}
        if kind == "cache":
            N = _log(rng, 16, 30000)
            B = _log(rng, 1, max(1, min(16, 4_000_000_00 // (N * Hkv * d * 8))))
            return dict(case, B=B, Nq=rng.choice([1, 1, 1, 2, 5, 13]), Nk=N, causal=True, lens=rng.random() < 0.6)
        N = _log(rng, 16, 6000)
        room = (150_000_000 if kind == "train" else 400_000_000) * 64 // d
        B = _log(rng, 1, max(1, min(8, room // (N * N * H))))
        if B * N * N * H > room:
            N = int(math.sqrt(room / (B * H)))
        Nq = N if rng.random() < 0.7 else max(1, N - rng.randint(0, N // 2))
        return dict(case, B=B, Nq=Nq, Nk=N, causal=rng.random() < 0.5, lens=rng.random() < 0.4)
    width = _log(rng, 48, 1000)
    layers = _log(rng, 1, max(1, min(12, 90_000_000 // (12 * width * width))))
    return {"op": op, "width": width, "layers": layers, "bits": rng.choice([8, 32]), "dtype": rng.choice(["f32", "f32", "bf16", "f16"])}


# ---- shapes ------------------------------------------------------------------------------------------------------------------
def _shapes(case):
    """a tower's parameters: the four matrices, their biases and the norms of every layer, and an odd-sized head"""
    w = case["width"]
    per = [(3 * w, w), (w, w), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,), (w,), (w,), (w,), (w,)]
    return per * case["layers"] + [(w + 1, 33), (7,), (1,)]


def _spans(case):
    """(offset, count, shape) of each parameter in a flat buffer, every one on a block's border; and the buffer's length"""
    spans, at = [], 0
    for s in _shapes(case):
        n = math.prod(s)
        spans.append((at, n, s))
        at += -(-n // BLOCK) * BLOCK
    return spans, at


def _lens(case):
    """valid keys of each batch entry: spread from none to all where `lens`, else all"""
    B, N = case["B"], case["Nk"]
    if not case["lens"]:
        return [N] * B
    if B == 1:
        return [max(1, (3 * N) // 4)]
    least = 0 if case["train"] else 1
    return [max(least, (N * i) // (B - 1)) for i in range(B)]


def _starts(case):
    """position of each batch entry's first query: behind what the cache holds, or 0 where a padded batch is trained"""
    if case["train"]:
        return [0] * case["B"]
    return [max(0, n - case["Nq"]) for n in _lens(case)]


def _pairs(case):
    """visible (query, key) pairs of one head, over the batch"""
    total = 0
    for n, s in zip(_lens(case), _starts(case)):
        if not case["causal"]:
            total += case["Nq"] * n
            continue
        full = max(0, min(case["Nq"], n - s))             # queries i with s + i + 1 <= n see s + i + 1 keys, the others n
        total += full * s + full * (full + 1) // 2 + (case["Nq"] - full) * n
    return total


def work(case):
    if case["op"] == "rotary":
        size = 4 if case["dtype"] == "f32" else 2
        n = case["B"] * case["N"] * (case["H"] + case["Hkv"]) * case["dh"]
        rot = 2 * (case["s0"] + case["s1"] + case["s2"])
        passes = 2 if case["train"] else 1
        pos = 12 * case["B"] * case["N"]
        return {"bytes": passes * (2 * n * size + pos), "flops": passes * 3 * n * rot // case["dh"]}
    if case["op"] == "diff":
        B, H, Hkv, d = case["B"], case["H"], case["Hkv"], case["d"]
        q = B * case["Nq"] * H * 2 * d * 2
        kv = sum(_lens(case)) * Hkv * 4 * d * 2
        if case["train"]:
            return {"bytes": 2 * (2 * q + kv), "flops": 28 * d * H * _pairs(case)}
        return {"bytes": 2 * q + kv, "flops": 8 * d * H * _pairs(case)}
    n = sum(s[1] for s in _spans(case)[0])
    p = 4 if case["dtype"] == "f32" else 2
    if case["bits"] == 32:
        return {"bytes": n * (3 * p + 16), "flops": 15 * n}
    return {"bytes": n * (3 * p + 4 + 4) + n // BLOCK * 16, "flops": 30 * n}      # the values of both moments are written too, in 16 bits


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _positions(case, g):
    """(slice, row, column) of each token: 0 for a class token, then a grid that is as near a cube as the count allows; `far` puts the
    sequence hundreds of thousands of steps from the origin on its first axis"""
    B, N = case["B"], case["N"]
    side = max(1, round((max(1, N - 1)) ** (1 / 3)))
    i = torch.arange(N, device=DEV).sub_(1).clamp_(min=0)
    grid = torch.stack([i // (side * side), i // side % side, i % side])
    pos = grid[:, None].repeat(1, B, 1)
    if case["far"]:
        pos[0] += torch.randint(1000, 800000, (B, 1), generator=g, device=DEV)
    else:
        pos += torch.randint(0, 4, (3, B, 1), generator=g, device=DEV)
    return pos.to(torch.int32)


def _quantise(m, v):
    """the 8-bit form of reals m and v >= 0 (whole blocks): codes and scales"""
    def parts(x):
        x = x.view(-1, BLOCK)
        s = x.abs().amax(1, keepdim=True)
        return s, torch.where(s > 0, x / s, torch.zeros_like(x))
    sm, rm = parts(m)
    sv, rv = parts(v.sqrt())
    cm = (rm.abs().sqrt() * 127).round() * rm.sign()
    cv = torch.maximum((rv.sqrt() * 255).round(), (rv > 0).to(rv.dtype))
    return cm.to(torch.int8).view(-1), cv.to(torch.uint8).view(-1), sm.float().view(-1), sv.float().view(-1)


def _values(cm, cv, sm, sv, dtype):
    """the values (m, sqrt v) that codes and scales stand for"""
    cm, cv = cm.view(-1, BLOCK).to(dtype), cv.view(-1, BLOCK).to(dtype)
    rm, rv = cm / 127, cv / 255
    return (sm.to(dtype)[:, None] * (rm * rm.abs())).view(-1), (sv.to(dtype)[:, None] * (rv * rv)).view(-1)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    if case["op"] == "rotary":
        B, N, H, Hkv, dh, dt = case["B"], case["N"], case["H"], case["Hkv"], case["dh"], DT[case["dtype"]]
        # one projection's output, as attention reads it: q, k and v heads side by side, q and k taken as views
        qkv = _rand(g, B, N, H + 2 * Hkv, dh, dtype=dt)
        st["q"], st["k"] = qkv[:, :, :H], qkv[:, :, H:H + Hkv]
        st["pos"] = _positions(case, g)
        if case["train"]:
            st["gq"], st["gk"] = _rand(g, B, N, H, dh, dtype=dt), _rand(g, B, N, Hkv, dh, dtype=dt)
            st["q"], st["k"] = st["q"].requires_grad_(), st["k"].requires_grad_()
        if own:
            from hsenet_amd import rotary
            st["plan"] = rotary.RotaryAxes((case["s0"], case["s1"], case["s2"]), theta=case["theta"], ladder=case["ladder"],
                                           interleaved=case["interleaved"], device=DEV)
        return st
    if case["op"] == "diff":
        B, H, Hkv, d, dt = case["B"], case["H"], case["Hkv"], case["d"], DT[case["dtype"]]
        st["q"] = _rand(g, B, case["Nq"], 2 * H, d, dtype=dt)
        st["k"] = _rand(g, B, case["Nk"], 2 * Hkv, d, dtype=dt)
        st["v"] = _rand(g, B, case["Nk"], Hkv, 2 * d, dtype=dt)
        st["lam"] = 0.2 + 0.6 * torch.rand(H, generator=g, device=DEV)
        st["len"] = torch.tensor(_lens(case), dtype=torch.int32, device=DEV)
        st["start"] = torch.tensor(_starts(case), dtype=torch.int32, device=DEV)
        if case["train"]:
            st["go"] = _rand(g, B, case["Nq"], H, 2 * d, dtype=dt)
            for n in ("q", "k", "v", "lam"):
                st[n].requires_grad_()
        return st
    spans, total = _spans(case)
    dt = DT[case["dtype"]]
    held = torch.zeros(total, device=DEV)
    for at, n, _ in spans:
        held[at:at + n] = 1.0
    st["p"] = (_rand(g, total, scale=0.02) * held).to(dt)
    st["g"] = (_rand(g, total, scale=1e-3) * held).to(dt)
    m, v = _rand(g, total, scale=3e-4) * held, (_rand(g, total, scale=1e-3) * held).square() * 0.5 + 1e-8 * held
    if case["bits"] == 8:
        st["cm"], st["cv"], st["sm"], st["sv"] = _quantise(m, v)
        st["m"], st["v"] = torch.zeros(total, dtype=torch.bfloat16, device=DEV), torch.zeros(total, dtype=torch.bfloat16, device=DEV)
    else:
        st["m"], st["v"] = m, v
    st["step"] = STEP0
    if own:
        from hsenet_amd import optim
        cut = lambda t: [t[at:at + n].view(s) for at, n, s in spans]  # noqa: E731
        ps = [x.requires_grad_() for x in cut(st["p"].detach())]
        for x, y in zip(ps, cut(st["g"])):
            x.grad = y
        opt = optim.AdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=case["bits"])
        if case["bits"] == 8:
            blocks = [(at // BLOCK, -(-n // BLOCK)) for at, n, _ in spans]
            for x, cm, cv, (b, k) in zip(ps, cut(st["cm"]), cut(st["cv"]), blocks):
                opt.set_state(x, step=STEP0, exp_avg=cm, exp_avg_sq=cv, exp_avg_scale=st["sm"][b:b + k], exp_avg_sq_scale=st["sv"][b:b + k])
            st["ms"], st["vs"] = cut(st["m"]), cut(st["v"])
        else:
            for x, y, z in zip(ps, cut(st["m"]), cut(st["v"])):
                opt.set_state(x, step=STEP0, exp_avg=y, exp_avg_sq=z)
        st["opt"] = opt
    return st


# ---- rotary ------------------------------------------------------------------------------------------------------------------
def _angles(case, pos, dtype=torch.float64):
    """angle of each (batch, token, pair), in 64 bits"""
    sections = (case["s0"], case["s1"], case["s2"])
    P = sum(sections)
    axis = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor(sections, device=DEV))
    j = torch.arange(P, device=DEV, dtype=dtype)
    if case["ladder"] == "per_axis":
        count = torch.tensor(sections, device=DEV, dtype=dtype)[axis]
        first = torch.tensor((0, sections[0], sections[0] + sections[1]), device=DEV, dtype=dtype)[axis]
        e = (j - first) / count
    else:
        e = j / P
    return pos.to(dtype)[axis].permute(1, 2, 0) * torch.pow(torch.tensor(case["theta"], device=DEV, dtype=dtype), -e)


def _turn(x, cos, sin, interleaved):
    """x with the pairs of its first 2 P columns turned"""
    P = cos.shape[-1]
    cos, sin = cos[:, :, None], sin[:, :, None]
    if interleaved:
        a, b = x[..., 0:2 * P:2], x[..., 1:2 * P:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :P], x[..., P:2 * P]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., 2 * P:]], -1)


def _rotary(st):
    case = st["case"]
    if own:
        from hsenet_amd import rotary
        if not case["train"]:
            return rotary.rotary_axes(st["q"], st["k"], st["pos"], st["plan"])
        with torch.enable_grad():
            q, k = rotary.rotary_axes(st["q"], st["k"], st["pos"], st["plan"])
            dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"]))
        return q.detach(), k.detach(), dq, dk
    ang = _angles(case, st["pos"])
    cos, sin = ang.cos().float(), ang.sin().float()
    out = [_turn(st[n].detach().float(), cos, sin, case["interleaved"]).to(st[n].dtype) for n in ("q", "k")]
    if case["train"]:
        out += [_turn(st[n].float(), cos, -sin, case["interleaved"]).to(st[n].dtype) for n in ("gq", "gk")]
    return tuple(out)


# ---- differential attention ----------------------------------------------------------------------------------------------------
def _hidden(case, st):
    """[B, 1, 1, Nq, Nk]: True where a query does not see a key"""
    j = torch.arange(case["Nk"], device=DEV)
    hide = (j[None, :] >= st["len"][:, None])[:, None, None, None, :]
    if case["causal"]:
        i = torch.arange(case["Nq"], device=DEV)
        hide = hide | (j[None, None, :] > (st["start"][:, None] + i[None, :])[:, :, None])[:, None, None]
    return hide


def _softmax(s, hide):
    """softmax over the visible keys; a row that sees none is zero"""
    s = s.masked_fill(hide, float("-inf"))
    e = (s - s.amax(-1, keepdim=True).clamp(min=torch.finfo(s.dtype).min)).exp()
    return e / e.sum(-1, keepdim=True).clamp(min=torch.finfo(s.dtype).tiny)


def _diff_plain(case, q, k, v, lam, hide):
    B, H, Hkv, d = case["B"], case["H"], case["Hkv"], case["d"]
    G = H // Hkv
    # heads in front, the query heads of a key head side by side: [B, Hkv, G, 2, N, d]
    q = q.float().view(B, case["Nq"], Hkv, G, 2, d).permute(4, 0, 2, 3, 1, 5)
    k = k.float().view(B, case["Nk"], Hkv, 1, 2, d).permute(4, 0, 2, 3, 1, 5)
    v = v.float().view(B, case["Nk"], Hkv, 1, 2 * d).permute(0, 2, 3, 1, 4)
    c = d ** -0.5
    p1 = _softmax(torch.matmul(q[0], k[0].transpose(-1, -2)) * c, hide)
    p2 = _softmax(torch.matmul(q[1], k[1].transpose(-1, -2)) * c, hide)
    o = torch.matmul(p1 - lam.view(1, Hkv, G, 1, 1) * p2, v)
    return o.permute(0, 3, 1, 2, 4).reshape(B, case["Nq"], H, 2 * d)


def _diff(st):
    case = st["case"]
    names = ("q", "k", "v", "lam")
    if own:
        from hsenet_amd.diff_attn import diff_attention
        kw = {"causal": case["causal"], "q_start": st["start"], "kv_len": st["len"] if case["lens"] else None}
        if not case["train"]:
            return diff_attention(st["q"], st["k"], st["v"], st["lam"], **kw)
        with torch.enable_grad():
            o = diff_attention(st["q"], st["k"], st["v"], st["lam"], **kw)
            grads = torch.autograd.grad(o, [st[n] for n in names], st["go"])
        return (o.detach(), *grads)
    hide = _hidden(case, st)
    if not case["train"]:
        return _diff_plain(case, st["q"], st["k"], st["v"], st["lam"], hide).to(st["q"].dtype)
    with torch.enable_grad():
        x = [st[n].detach().float().requires_grad_() for n in names]
        o = _diff_plain(case, *x, hide)
        grads = torch.autograd.grad(o, x, st["go"].float())
    return (o.detach().to(st["q"].dtype), *[t.to(st[n].dtype) for t, n in zip(grads, names)])


# ---- AdamW -------------------------------------------------------------------------------------------------------------------
def _adamw(st):
    case = st["case"]
    if own:
        st["opt"].step()
        if case["bits"] == 8:
            st["opt"].read_moments(st["ms"], st["vs"])
        return st["p"], st["m"], st["v"]
    st["step"] += 1
    c1, c2 = 1 - B1 ** st["step"], math.sqrt(1 - B2 ** st["step"])
    if case["bits"] == 8:
        m, u = _values(st["cm"], st["cv"], st["sm"], st["sv"], torch.float32)
        v = u * u
    else:
        m, v = st["m"], st["v"]
    g = st["g"].float()
    m = m * B1 + g * (1 - B1)
    v = v * B2 + (g * g) * (1 - B2)
    p = st["p"].float() * (1 - LR * WD) - (LR / c1) * m / (v.sqrt() / c2 + EPS)
    st["p"].copy_(p)
    if case["bits"] == 8:
        st["cm"], st["cv"], st["sm"], st["sv"] = _quantise(m, v)
        m, u = _values(st["cm"], st["cv"], st["sm"], st["sv"], torch.float32)
        v = u * u
    st["m"].copy_(m)
    st["v"].copy_(v)
    return st["p"], st["m"], st["v"]


def run(state):
    op = state["case"]["op"]
    with torch.no_grad():
        return _rotary(state) if op == "rotary" else _diff(state) if op == "diff" else _adamw(state)


# ---- 64 bits -----------------------------------------------------------------------------------------------------------------
def _exact_rotary(case, st):
    sections = [case["s0"], case["s1"], case["s2"]]
    freq, axis = [], []
    for a, n in enumerate(sections):
        for i in range(n):
            e = i / n if case["ladder"] == "per_axis" else len(freq) / sum(sections)
            freq.append(case["theta"] ** -e)
            axis.append(a)
    f, P = torch.tensor(freq, dtype=torch.float64, device=DEV), len(freq)
    w = torch.exp(1j * (st["pos"][axis].double().movedim(0, -1) * f))[:, :, None]

    def turned(x, w):
        y = x.detach().double().clone()
        lo, hi = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if case["interleaved"] else (slice(0, P), slice(P, 2 * P))
        z = torch.complex(y[..., lo], y[..., hi]) * w
        y[..., lo], y[..., hi] = z.real, z.imag
        return y
    out = [turned(st["q"], w), turned(st["k"], w)]
    if case["train"]:
        out += [turned(st["gq"], w.conj()), turned(st["gk"], w.conj())]
    return tuple(out)


def _exact_diff(case, st):
    B, H, Hkv, d, Nq = case["B"], case["H"], case["Hkv"], case["d"], case["Nq"]
    q, k, v, lam = (st[n].detach().double() for n in ("q", "k", "v", "lam"))
    go = st["go"].double() if case["train"] else None
    o, dq, dk, dv, dlam = torch.zeros(B, Nq, H, 2 * d, dtype=torch.float64, device=DEV), q * 0, k * 0, v * 0, lam * 0
    c, rows = 1 / math.sqrt(d), 2048
    for b, (n, start) in enumerate(zip(_lens(case), _starts(case))):
        if n == 0:
            continue
        at = torch.arange(n, device=DEV)
        for h in range(H):
            g = h // (H // Hkv)
            V = v[b, :n, g]
            for r in range(0, Nq, rows):
                i = slice(r, min(Nq, r + rows))
                seen = torch.ones(i.stop - r, n, dtype=torch.bool, device=DEV)
                if case["causal"]:
                    seen = at[None] <= start + torch.arange(r, i.stop, device=DEV)[:, None]
                maps = []
                for m in (0, 1):
                    s = (q[b, i, 2 * h + m] @ k[b, :n, 2 * g + m].T) * c
                    s = torch.where(seen, s, -math.inf)
                    maps.append(torch.softmax(s, -1).nan_to_num(0.0))
                o[b, i, h] = maps[0] @ V - lam[h] * (maps[1] @ V)
                if go is None:
                    continue
                G = go[b, i, h]
                dv[b, :n, g] += (maps[0] - lam[h] * maps[1]).T @ G
                dP = G @ V.T
                for m, w in ((0, 1.0), (1, -lam[h])):
                    D = (maps[m] * dP).sum(-1, keepdim=True)
                    if m:
                        dlam[h] -= D.sum()
                    dS = maps[m] * (dP - D) * (w * c)
                    dq[b, i, 2 * h + m] = dS @ k[b, :n, 2 * g + m]
                    dk[b, :n, 2 * g + m] += dS.T @ q[b, i, 2 * h + m]
    return o if go is None else (o, dq, dk, dv, dlam)


def _exact_adamw(case, st):
    g, t, p = st["g"].double(), STEP0 + 1, st["p"].double()
    if case["bits"] == 8:
        a, b = st["cm"].double() / 127, st["cv"].double() / 255
        m = a * a.abs() * st["sm"].double().repeat_interleave(BLOCK)
        v = (b * b * st["sv"].double().repeat_interleave(BLOCK)).square()
    else:
        m, v = st["m"].double(), st["v"].double()
    m = torch.lerp(g, m, B1)
    v = torch.lerp(g.square(), v, B2)
    hat_m, hat_v = m / (1 - B1 ** t), v / (1 - B2 ** t)
    p = p - LR * (hat_m / (hat_v.sqrt() + EPS) + WD * p)
    if case["bits"] == 8:
        # a code is the nearest whole number to 127 (255) times the root of the share of the block's largest, and a scale is held in 32 bits
        u = v.sqrt()
        sm = m.unflatten(0, (-1, BLOCK)).abs().max(1).values.float().double().clamp(min=1e-300).repeat_interleave(BLOCK)
        su = u.unflatten(0, (-1, BLOCK)).max(1).values.float().double().clamp(min=1e-300).repeat_interleave(BLOCK)
        a = torch.round(torch.sqrt(m.abs() / sm) * 127) / 127
        b = torch.round(torch.sqrt(u / su) * 255)
        b = torch.where((u > 0) & (b < 1), 1.0, b) / 255
        m, v = torch.copysign(a * a * sm, m), (b * b * su).square()
    return p, m, v


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "diff": _exact_diff, "adamw": _exact_adamw}[case["op"]](case, st)
