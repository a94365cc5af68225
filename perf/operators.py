"""The conditioning operators of the video and image transformers as measurable cases.

Three operators: attention of latent tokens to an encoder's states of another length (`cross_attention`), attention of a
batch whose samples share a long run of cached keys (`prefix_attention`), and the row kernel between two sub-layers of a
sandwich-norm block (`rmsnorm_gate_residual_modulate`). With `own` false every case runs in elementary torch operations;
with `own` true it makes the calls of the public entry points. `exact` is the definition in 64 bits.

    cross_attention   o[b,i,h] = sum_j p_j v[b,j,h'],  p = softmax over the keys j that sample b may see of scale q.k_j
    prefix_attention  the same over the keys of the shared prefix followed by the sample's own keys
    rmsnorm_gate_residual_modulate
                      x = res + g (y / rms(y)) w   (g = gate or tanh(gate); the normalisation of y is optional)
                      h = (x / rms(x)) w' (1 + scale) + shift, of x as it is stored

A query without a visible key gives zeros, and -inf as its log-sum-exp. h' = h // (heads / key heads).
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------------------------
def _cross(name, layout, dtype, B, Sq, H, Hkv, D, Skv, least, lse):
    """layout: "dense" (every sample sees all Skv states), "padded" (the first len of Skv), "packed" (the samples' states
    in one row after the other) or "masked" (a truth value per state; the padding is on the left). `least`: the shortest
    sample's length; the others are spread between it and Skv."""
    return {"name": name, "op": "cross", "layout": layout, "dtype": dtype, "B": B, "Sq": Sq, "H": H, "Hkv": Hkv, "D": D,
            "Skv": Skv, "least": least, "lse": lse}  # fmt: skip


def _prefix(name, dtype, B, Sq, H, Hkv, D, P, S, least, lse):
    return {"name": name, "op": "prefix", "dtype": dtype, "B": B, "Sq": Sq, "H": H, "Hkv": Hkv, "D": D, "P": P, "S": S,
            "least": least, "lse": lse}  # fmt: skip


def _norm(name, dtype, B, S, C, tables, post, tanh):
    """tables: "sample" (one row of gate / shift / scale per sample) or "token" (one per token)."""
    return {"name": name, "op": "norm", "dtype": dtype, "B": B, "S": S, "C": C, "tables": tables, "post": post, "tanh": tanh}


def listed():
    return [
        # one new token of each of eight streams against its own prompt
        _cross("cross_one_token", "padded", "fp16", 8, 1, 16, 16, 64, 512, 1, False),
        # every latent frame attends to the audio tokens of its moment (frames are the batch)
        _cross("cross_frames_to_audio", "dense", "bf16", 21, 1560, 40, 40, 128, 32, 32, False),
        # a 480p clip under guidance: prompt and negative prompt, their valid states packed
        _cross("cross_clip_to_prompts", "packed", "bf16", 2, 37440, 32, 32, 128, 512, 183, False),
        # left-padded prompts kept in place, an odd number of latent tokens
        _cross("cross_masked_prompts", "masked", "fp16", 2, 6143, 32, 32, 64, 1024, 77, True),
        # a handful of summary tokens reads a long encoding
        _cross("cross_few_to_long", "dense", "bf16", 1, 5, 32, 8, 128, 131072, 131072, True),
        # a short request: a few tokens each, one sample without states of its own
        _prefix("prefix_short", "fp16", 3, 4, 8, 2, 64, 77, 33, 0, True),
        # both guidance branches continue a clip whose clean frames' keys are cached once
        _prefix("prefix_clip_continuation", "bf16", 2, 3120, 32, 32, 128, 9360, 3120, 3120, False),
        # many streams of one scene, one token each
        _prefix("prefix_many_streams", "bf16", 64, 1, 32, 8, 128, 16384, 1000, 0, False),
        # three rows: the smallest call
        _norm("norm_three_rows", "bf16", 1, 3, 2048, "sample", True, True),
        # an image with its caption, two branches
        _norm("norm_image", "bf16", 2, 4224, 3840, "sample", True, True),
        # a long clip
        _norm("norm_clip", "bf16", 1, 37441, 2048, "sample", True, True),
        # tokens with time steps of their own: tables per token, no norm behind the sub-layer
        _norm("norm_token_tables", "fp16", 2, 3001, 4096, "token", False, False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cross", "cross", "prefix", "norm"])
    if op == "norm":
        C = 8 * _log(rng, 16, 1024)
        B = rng.choice([1, 1, 2, 3])
        S = _log(rng, 1, 40000 * 2048 // C // B)
        tables = rng.choice(["sample", "sample", "token"])
        if tables == "token":
            S = max(1, S // 4)
        return _norm("", rng.choice(["bf16", "bf16", "fp16", "fp32"]), B, S, C, tables, rng.random() < 0.7, rng.random() < 0.5)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    D = rng.choice([64, 128, 128, 128, 40, 72, 96])
    Hkv = rng.choice([1, 2, 4, 8, 16])
    H = Hkv * rng.choice([1, 1, 2, 3, 4, 8]) if Hkv < 16 else Hkv * rng.choice([1, 2])
    few = rng.random() < 0.4
    B = _log(rng, 1, 64 if few else 8)
    Sq = _log(rng, 1, 16) if few else _log(rng, 17, 20000)
    pairs = 4e11 / (4 * B * H * Sq * D)  # keys that keep the work under the largest listed case's
    scores = 8e8 / (B * H * Sq)
    rows = 3e8 / (B * Hkv * D)
    most = max(1, int(min(pairs, scores, rows, 100000 if few else 8192)))
    if op == "cross":
        Skv = _log(rng, 1, most)
        layout = rng.choice(["dense", "padded", "packed", "masked"])
        least = Skv if layout == "dense" else rng.choice([0, 1, max(1, Skv // 2)])
        return _cross("", layout, dtype, B, Sq, H, Hkv, D, Skv, min(least, Skv), rng.random() < 0.5)
    S = _log(rng, 1, max(1, most // 4))
    return _prefix("", dtype, B, Sq, H, Hkv, D, _log(rng, 1, max(1, most - S)), S, rng.choice([S, 0, 1]), rng.random() < 0.5)


def _lens(case):
    """The samples' numbers of states: between `least` and the most, in no order, part of the case."""
    B, most, least = case["B"], case["Skv"] if case["op"] == "cross" else case["S"], case["least"]
    if B == 1:
        return [most]
    return [least + (most - least) * ((5 * b + 3) % B) // (B - 1) if B % 5 else least + (most - least) * b // (B - 1) for b in range(B)]


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1_000_003 * int(seed) + 17)
    dt = _TYPES[case["dtype"]]

    def normal(*shape, dtype=dt, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    st = {"op": case["op"], "case": case}
    if case["op"] == "norm":
        B, S, C = case["B"], case["S"], case["C"]
        n = S if case["tables"] == "token" else 1
        f32 = dict(dtype=torch.float32)
        st |= dict(res=normal(B, S, C, std=2.0), y=normal(B, S, C), weight=1 + normal(C, std=0.1) if case["post"] else None,
                   gate=normal(B, n, C, std=0.5, **f32), next_weight=1 + normal(C, std=0.1),
                   shift=normal(B, n, C, std=0.3, **f32), scale=normal(B, n, C, std=0.3, **f32))  # fmt: skip
        return st
    B, Sq, H, Hkv, D = (case[n] for n in ("B", "Sq", "H", "Hkv", "D"))
    lens = _lens(case)
    st["q"] = normal(B, Sq, H, D)  # q and k leave a norm over the head, v a projection with a mean of its own
    mean = normal(Hkv, D, dtype=torch.float32, std=0.5)
    if case["op"] == "prefix":
        P, S = case["P"], case["S"]
        st |= dict(k_prefix=normal(1, P, Hkv, D), v_prefix=(normal(1, P, Hkv, D, dtype=torch.float32) + mean).to(dt),
                   k=normal(B, S, Hkv, D), v=(normal(B, S, Hkv, D, dtype=torch.float32) + mean).to(dt))  # fmt: skip
        st["kv_lens"] = None if case["least"] == S else torch.tensor(lens, dtype=torch.int32, device="cuda")
        return st
    Skv, layout = case["Skv"], case["layout"]
    if layout == "packed":
        T = sum(lens)
        st |= dict(k=normal(T, Hkv, D), v=(normal(T, Hkv, D, dtype=torch.float32) + mean).to(dt), longest=max(lens))
        st["cu_kv"] = torch.tensor([sum(lens[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
        return st
    st |= dict(k=normal(B, Skv, Hkv, D), v=(normal(B, Skv, Hkv, D, dtype=torch.float32) + mean).to(dt))
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if layout == "padded":
        st["kv_lens"] = n
    elif layout == "masked":
        st["key_mask"] = torch.arange(Skv, device="cuda")[None] >= Skv - n[:, None]
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(st):
    return _run_own(st) if own else {"cross": _plain_cross, "prefix": _plain_prefix, "norm": _plain_norm}[st["op"]](st)


def _run_own(st):
    from telefuser_b200.ops import context_attention as CA
    from telefuser_b200.ops import functional as TF

    case = st["case"]
    if st["op"] == "norm":
        return TF.rmsnorm_gate_residual_modulate(st["res"], st["y"], st["weight"], st["gate"], st["next_weight"], st["shift"],
                                                 st["scale"], eps=1e-6, tanh_gate=case["tanh"], post_norm=case["post"])  # fmt: skip
    if st["op"] == "prefix":
        return CA.prefix_attention(st["q"], st["k_prefix"], st["v_prefix"], st["k"], st["v"], kv_lens=st["kv_lens"],
                                   return_lse=case["lse"])  # fmt: skip
    return CA.cross_attention(st["q"], st["k"], st["v"], kv_lens=st.get("kv_lens"), cu_kv=st.get("cu_kv"),
                              key_mask=st.get("key_mask"), return_lse=case["lse"])  # fmt: skip


def _plain_softmax(s, visible):
    """Weights and log-sum-exp over the last axis of s where `visible`; rows that see nothing: zeros and -inf."""
    s = s.masked_fill(~visible, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > float("-inf"), m, torch.zeros_like(m)))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total)), (torch.log(total) + m).squeeze(-1)


def _plain_cross(st):
    case, q, k, v = st["case"], st["q"].float(), st["k"].float(), st["v"].float()
    B, Sq, H, D = q.shape
    if "cu_kv" in st:
        cu = st["cu_kv"].long()
        j = torch.arange(st["longest"], device=q.device)[None]
        visible = j < (cu[1:] - cu[:-1])[:, None]
        at = (cu[:-1, None] + j).clamp(max=k.shape[0] - 1)
        k, v = k[at], v[at]
    elif "kv_lens" in st:
        visible = torch.arange(k.shape[1], device=q.device)[None] < st["kv_lens"][:, None]
    else:
        visible = st.get("key_mask")
        visible = torch.ones(B, k.shape[1], dtype=torch.bool, device=q.device) if visible is None else visible
    Hkv = k.shape[2]
    qg = (q * (1.0 / math.sqrt(D))).reshape(B, Sq, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    s = qg @ k.permute(0, 2, 3, 1)  # [B, Hkv, G Sq, Skv]
    p, lse = _plain_softmax(s, visible[:, None, None])
    v = torch.where(visible[:, :, None, None], v, torch.zeros_like(v))
    o = (p @ v.transpose(1, 2)).reshape(B, H, Sq, D).transpose(1, 2).to(_TYPES[case["dtype"]])
    return (o, lse.reshape(B, H, Sq)) if case["lse"] else o


def _plain_prefix(st):
    case, q = st["case"], st["q"].float()
    B, Sq, H, D = q.shape
    kp, vp, k, v = (st[n].float() for n in ("k_prefix", "v_prefix", "k", "v"))
    Hkv, P, S = k.shape[2], kp.shape[1], k.shape[1]
    qg = (q * (1.0 / math.sqrt(D))).reshape(B, Sq, Hkv, H // Hkv, D).permute(2, 0, 3, 1, 4)  # [Hkv, B, G, Sq, D]
    rows = (H // Hkv) * Sq
    sp = qg.reshape(Hkv, B * rows, D) @ kp[0].permute(1, 2, 0)  # the prefix against all samples' rows at once
    so = qg.reshape(Hkv, B, rows, D) @ k.permute(2, 0, 3, 1)
    seen = torch.arange(S, device=q.device)[None]
    seen = seen < (seen.new_full((B,), S) if st["kv_lens"] is None else st["kv_lens"])[:, None]
    visible = torch.cat([seen.new_ones(B, P), seen], dim=1)[None, :, None]
    p, lse = _plain_softmax(torch.cat([sp.reshape(Hkv, B, rows, P), so], dim=-1), visible)
    o = (p[..., :P].reshape(Hkv, B * rows, P) @ vp[0].transpose(0, 1)).reshape(Hkv, B, rows, D)
    o = o + p[..., P:] @ torch.where(seen[:, :, None, None], v, torch.zeros_like(v)).permute(2, 0, 1, 3)
    o = o.reshape(Hkv, B, H // Hkv, Sq, D).permute(1, 3, 0, 2, 4).reshape(B, Sq, H, D).to(_TYPES[case["dtype"]])
    return (o, lse.reshape(Hkv, B, H // Hkv, Sq).permute(1, 0, 2, 3).reshape(B, H, Sq)) if case["lse"] else o


def _plain_norm(st):
    case, y = st["case"], st["y"].float()
    if case["post"]:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * st["weight"].float()
    g = torch.tanh(st["gate"]) if case["tanh"] else st["gate"]
    x = (st["res"].float() + g * y).to(_TYPES[case["dtype"]])
    xf = x.float()
    h = xf / torch.sqrt((xf * xf).mean(-1, keepdim=True) + 1e-6) * st["next_weight"].float()
    return x, (h * (1 + st["scale"]) + st["shift"]).to(x.dtype)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    B = case["B"]
    if case["op"] == "norm":
        n = B * case["S"] * case["C"]
        tables = 3 * 4 * (n if case["tables"] == "token" else B * case["C"]) + 2 * e * case["C"]
        return {"bytes": 4 * n * e + tables, "flops": 12 * n}
    Sq, H, Hkv, D = (case[k] for k in ("Sq", "H", "Hkv", "D"))
    lens = _lens(case)
    out = 2 * B * Sq * H * D * e + (4 * B * H * Sq if case["lse"] else 0)
    if case["op"] == "prefix":
        return {"bytes": out + 2 * (case["P"] + sum(lens)) * Hkv * D * e, "flops": 4 * Sq * H * D * (B * case["P"] + sum(lens))}
    marks = B * case["Skv"] if case["layout"] == "masked" else 0
    return {"bytes": out + 2 * sum(lens) * Hkv * D * e + marks, "flops": 4 * Sq * H * D * sum(lens)}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, st)
    B, Sq, H, D = st["q"].shape
    lens = _lens(case)
    out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, Sq), float("-inf"), dtype=torch.float64, device="cuda")
    first = 0
    for b in range(B):
        n = lens[b]
        if case["op"] == "prefix":
            k = torch.cat([st["k_prefix"][0], st["k"][b, :n]])
            v = torch.cat([st["v_prefix"][0], st["v"][b, :n]])
        elif case["layout"] == "packed":
            k, v = st["k"][first : first + n], st["v"][first : first + n]
            first += n
        elif case["layout"] == "masked":
            k, v = st["k"][b, case["Skv"] - n :], st["v"][b, case["Skv"] - n :]
        else:
            k, v = st["k"][b, :n], st["v"][b, :n]
        if k.shape[0] == 0:
            continue
        for h in range(H):
            kh, vh = (t[:, h * case["Hkv"] // H].double() for t in (k, v))
            s = torch.einsum("id,jd->ij", st["q"][b, :, h].double(), kh) / D**0.5
            lse[b, h] = torch.logsumexp(s, dim=1)
            out[b, :, h] = torch.softmax(s, dim=1) @ vh
    return (out, lse) if case["lse"] else out


def _exact_norm(case, st):
    dt = _TYPES[case["dtype"]]
    res, y = st["res"].double(), st["y"].double()
    if case["post"]:
        y = st["weight"].double() * y * torch.rsqrt(y.square().mean(dim=-1, keepdim=True) + 1e-6)
    gate = st["gate"].double()
    x = torch.addcmul(res, gate.tanh() if case["tanh"] else gate, y)
    held = x.to(dt).double()
    h = st["next_weight"].double() * held * torch.rsqrt(held.square().mean(dim=-1, keepdim=True) + 1e-6)
    return x, h + h * st["scale"].double() + st["shift"].double()
