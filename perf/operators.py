"""Position rotation, the paged KV cache and the attention that reads it: cases and plain forms.

Four operators that a serving or training loop runs next to the dense attention:

* ``rope``    rotation of queries and keys by their positions (one axis, or several for images
              and video), and its gradient, which is the rotation by the opposite angle;
* ``append``  new keys and values written into their pages, keys (and queries) rotated on the way;
* ``paged``   attention of each sequence's newest tokens over its pages: one token per sequence,
              a few (speculative decoding), or whole chunks of a prompt;
* ``prefix``  the same for a batch whose sequences share one long prefix, read once for all.

``run`` computes them with elementary torch operations in 32 bits, or, with ``own`` set, through
the ``lvb`` package. ``exact`` computes them once more from their definitions in 64 bits.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


def _rope(name, B, Hq, Hkv, S, D, rot, axes, layout, dtype, inverse):
    return dict(name=name, op="rope", B=B, Hq=Hq, Hkv=Hkv, S=S, D=D, rot=rot, axes=axes,
                layout=layout, dtype=dtype, inverse=inverse)


def _append(name, B, Hq, Hkv, D, page, q_lo, q_hi, ctx_lo, ctx_hi, rot, axes, layout, dtype, shape):
    return dict(name=name, op="append", B=B, Hq=Hq, Hkv=Hkv, D=D, page=page, q_lo=q_lo, q_hi=q_hi,
                ctx_lo=ctx_lo, ctx_hi=ctx_hi, rot=rot, axes=axes, layout=layout, dtype=dtype,
                shape=shape)


def _paged(name, B, Hq, Hkv, D, page, q_lo, q_hi, ctx_lo, ctx_hi, dtype, shape, prefix=0):
    return dict(name=name, op="prefix" if prefix else "paged", B=B, Hq=Hq, Hkv=Hkv, D=D, page=page,
                q_lo=q_lo, q_hi=q_hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi, dtype=dtype, shape=shape,
                prefix=prefix)


def listed():
    return [
        # Queries and keys of the benchmark's fp16 attention (batch 4, 32 heads, 4,096 positions)
        # before that attention: the forward rotation of a training step or a prefill.
        _rope("rope_fwd_4096", 4, 32, 32, 4096, 128, 128, 1, "halves", "fp16", False),
        # Gradients of a video clip's queries and keys: time, height and width, an odd number of
        # patches, a quarter of each head not rotated, grouped key heads.
        _rope("rope_grad_video", 2, 16, 4, 5 * 23 * 37, 128, 96, 3, "pairs", "bf16", True),
        # One decoding step of the benchmark's grouped-query model: a token per sequence.
        _append("append_step", 8, 64, 8, 128, 64, 1, 1, 16384, 16384, 128, 1, "halves", "bf16", 1),
        # Prompts of very different length entering the cache together, image positions.
        _append("append_prompts", 9, 32, 8, 64, 16, 1, 4099, 0, 900, 64, 3, "halves", "fp16", 2),
        # A single user's short chat: the smallest call, where latency counts.
        _paged("decode_single", 1, 32, 8, 128, 16, 1, 1, 777, 777, "fp16", 3),
        # The benchmark's grouped-query KV cache (8 x 8 heads x 16,384), one new token each.
        _paged("decode_16384", 8, 64, 8, 128, 64, 1, 1, 16384, 16384, "bf16", 4),
        # A server's mixed batch: lengths from a few tokens to 30,000.
        _paged("decode_ragged", 61, 32, 4, 128, 32, 1, 1, 1, 30000, "bf16", 5),
        # Four drafted tokens per sequence to be verified, 64-wide heads.
        _paged("decode_draft", 24, 16, 8, 64, 128, 4, 4, 100, 9000, "fp16", 6),
        # Chunks of prompts behind what the cache holds already, with decoding tokens among them.
        _paged("chunked_prefill", 6, 32, 8, 128, 64, 1, 2048, 2000, 8000, "bf16", 5),
        # A few samples of one short prompt.
        _paged("prefix_samples", 4, 32, 8, 128, 16, 1, 1, 1, 64, "fp16", 8, prefix=500),
        # 64 users behind one long system prompt (the benchmark's 16,384 positions).
        _paged("prefix_16384", 64, 64, 8, 128, 64, 1, 1, 1, 2048, "bf16", 9, prefix=16384),
        # Drafted tokens behind a shared prefix that ends inside a page, one key head per head.
        _paged("prefix_draft", 32, 8, 8, 64, 32, 3, 3, 3, 300, "bf16", 10, prefix=4099),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "paged", "paged", "prefix"])
    dtype = rng.choice(["fp16", "bf16"])
    D = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 3, 4, 6, 8])
    layout = rng.choice(["halves", "pairs"])
    rot = rng.choice([D // 2, 3 * D // 4, D])
    axes = rng.choice([1, 1, 2, 3])
    page = rng.choice([8, 16, 32, 48, 64, 128, 256])
    shape = rng.randrange(1, 1 << 20)
    if op == "rope":
        B = _log(rng, 1, 8)
        # as many values at most as the largest listed rotation has
        S = _log(rng, 1, min(16384, 67108864 // (B * (Hq + Hkv) * D)))
        c = _rope("", B, Hq, Hkv, S, D, rot, axes, layout, rng.choice([dtype, dtype, "fp32"]),
                  rng.random() < 0.5)
    elif op == "append":
        B = _log(rng, 1, 64)
        q_hi = _log(rng, 1, max(1, min(4099, 16384 // B)))
        c = _append("", B, Hq, Hkv, D, page, rng.choice([1, q_hi]), q_hi, 0, _log(rng, 1, 4000), rot,
                    axes, layout, dtype, shape)
    elif op == "paged":
        B = _log(rng, 1, 64)
        if rng.random() < 0.7:      # decoding
            q_hi = rng.choice([1, 1, 2, 5])
            ctx = _log(rng, q_hi, min(60000, 8 * 60000 // (B * Hkv)))
            q_lo = 1 if rng.random() < 0.5 else q_hi
        else:                       # chunks
            B = min(B, 5)
            q_hi = _log(rng, 6, 2048)
            ctx = _log(rng, q_hi, 6000)
            q_lo = 1
        c = _paged("", B, Hq, Hkv, D, page, q_lo, q_hi, 1, max(1, ctx), dtype, shape)
    else:
        B = _log(rng, 2, 64)
        prefix = _log(rng, 100, 16384)
        q = rng.choice([1, 1, 1, 2, 3])
        c = _paged("", B, Hq, Hkv, D, page, q, q, q, _log(rng, q, 2048), dtype, shape, prefix=prefix)
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, cached tokens) of each sequence: of the case alone, not of the seed. A paged
    or prefix case's second number counts the new tokens too."""
    r = random.Random(case["shape"])
    q, n = [], []
    for _ in range(case["B"]):
        qi = _log(r, case["q_lo"], case["q_hi"])
        if case["op"] == "append":
            ni = r.randint(case["ctx_lo"], case["ctx_hi"]) + qi
        else:
            ni = max(qi, _log(r, max(case["ctx_lo"], 1), case["ctx_hi"]))
        q.append(qi)
        n.append(ni)
    return q, n


def _sections(case):
    half = case["rot"] // 2
    a = case["axes"]
    rest = half // a
    return [half - rest * (a - 1)] + [rest] * (a - 1)


def _freqs(case):
    half = case["rot"] // 2
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    return torch.exp(-math.log(10000.0) * i / half)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DT[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=g).to(dt)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, device="cuda", dtype=torch.int32, generator=g)

    Hq, Hkv, D, B = case["Hq"], case["Hkv"], case["D"], case["B"]
    s = dict(case=dict(case), call=None)
    if case["op"] == "rope":
        S, axes = case["S"], case["axes"]
        s["Q"], s["K"] = randn(B, Hq, S, D), randn(B, Hkv, S, D)
        s["Qo"], s["Ko"] = torch.empty_like(s["Q"]), torch.empty_like(s["K"])
        if axes == 1:               # each sequence starts somewhere of its own
            s["pos"] = (ints(0, 100000, 1, B, 1)
                        + torch.arange(S, device="cuda", dtype=torch.int32))
        else:
            s["pos"] = ints(0, 4096, axes, B, S)
        s["freqs"], s["sections"] = _freqs(case), _sections(case)
        return s
    q, n = _lengths(case)
    page, T = case["page"], sum(q)
    per = max(-(-x // page) for x in n)
    prefix = case.get("prefix", 0)
    per_prefix = -(-prefix // page)
    used = sum(-(-x // page) for x in n) + per_prefix
    num_pages = used + used // 8 + 1
    order = torch.randperm(num_pages, device="cuda", generator=g).to(torch.int32)
    # Each sequence's pages lie anywhere in the cache; what its row has behind them is no page.
    counts = torch.tensor([-(-x // page) for x in n])
    first = (torch.cumsum(counts, 0) - counts).cuda()[:, None]
    col = torch.arange(per, device="cuda")[None, :]
    inside = col < counts.cuda()[:, None]
    table = torch.where(inside, order[(first + col).clamp(max=num_pages - 1)].long(), -1)
    s["table"] = table.to(torch.int32).contiguous()
    s["prefix_table"] = order[used - per_prefix:used].contiguous()
    s["lens"] = torch.tensor(n, dtype=torch.int32).cuda()
    s["cu"] = torch.tensor([0] + list(torch.cumsum(torch.tensor(q), 0)), dtype=torch.int32).cuda()
    s["max_q"], s["max_len"] = max(q), max(n)
    s["Kc"], s["Vc"] = randn(num_pages, page, Hkv, D), randn(num_pages, page, Hkv, D)
    s["Q"] = randn(T, Hq, D)
    if case["op"] == "append":
        s["K"], s["V"] = randn(T, Hkv, D), randn(T, Hkv, D)
        s["Qo"] = torch.empty_like(s["Q"])
        s["pos"] = ints(0, 100000, case["axes"], T) if case["axes"] > 1 else None
        s["freqs"], s["sections"] = _freqs(case), _sections(case)
    else:
        s["O"] = torch.empty_like(s["Q"])
        s["lse"] = torch.empty(T, Hq, device="cuda")
    return s


# ---- the framework's calls ----------------------------------------------------------------
def _lvb():
    p = str(Path("lava.jl_b200").resolve())
    if p not in sys.path:
        sys.path.insert(0, p)
    import lvb
    return lvb


def _run_own(s):
    # The buffers of a loop stay where they are: the call is described at its first pass.
    c = s["case"]
    if s["call"] is None:
        lvb = _lvb()
        if c["op"] == "rope":
            s["call"] = lvb.prepare_rope(s["Qo"], s["Q"], s["pos"], s["freqs"], Ko=s["Ko"], K=s["K"],
                                         sections=s["sections"], layout=c["layout"],
                                         inverse=c["inverse"])
        elif c["op"] == "append":
            s["call"] = lvb.prepare_kv_append(s["Kc"], s["Vc"], s["K"], s["V"], s["table"], s["lens"],
                                              cu_q=s["cu"], max_q=s["max_q"], Qo=s["Qo"], Q=s["Q"],
                                              pos=s["pos"], freqs=s["freqs"],
                                              sections=s["sections"], layout=c["layout"])
        else:
            more = {}
            if c["prefix"]:
                more = dict(prefix_table=s["prefix_table"], prefix_len=c["prefix"])
            s["call"] = lvb.prepare_attention_paged(s["O"], s["Q"], s["Kc"], s["Vc"], s["table"],
                                                    s["lens"], cu_q=s["cu"], max_q=s["max_q"],
                                                    lse=s["lse"], **more)
    s["call"]()
    if c["op"] == "rope":
        return s["Qo"], s["Ko"]
    if c["op"] == "append":
        return s["Kc"], s["Vc"], s["Qo"]
    return s["O"], s["lse"]


# ---- plain forms --------------------------------------------------------------------------
def _angles(pos, freqs, sections):
    """cos and sin [..., pairs] of positions [axes, ...]: each pair turns with its section's axis.
    The product is taken in 64 bits: a far position's angle has no digits left in 32."""
    axis = torch.repeat_interleave(torch.arange(len(sections), device=pos.device),
                                   torch.tensor(sections, device=pos.device),
                                   output_size=sum(sections))
    a = pos[axis].movedim(0, -1).double() * freqs
    return torch.cos(a).float(), torch.sin(a).float()


def _rotate(x, cos, sin, layout):
    """x [..., D] in 32 bits, its first 2·pairs elements rotated."""
    half = cos.shape[-1]
    r, rest = x[..., :2 * half].float(), x[..., 2 * half:].float()
    if layout == "halves":
        a, b = r[..., :half], r[..., half:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([r, rest], -1).to(x.dtype)


def _token_places(s):
    """Per token: its sequence and its place in that sequence's cache."""
    T = s["Q"].shape[0]
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["cu"][1:].contiguous(), t, right=True)
    return b, s["lens"][b] - (s["cu"][b + 1] - t)


def _plain_append(s):
    c = s["case"]
    b, place = _token_places(s)
    pos = s["pos"] if s["pos"] is not None else place[None, :]
    cos, sin = _angles(pos, s["freqs"], s["sections"])
    cos, sin = cos[:, None, :], sin[:, None, :]
    pages = s["table"][b, place // c["page"]].long()
    slots = (place % c["page"]).long()
    s["Kc"][pages, slots] = _rotate(s["K"], cos, sin, c["layout"])
    s["Vc"][pages, slots] = s["V"]
    s["Qo"].copy_(_rotate(s["Q"], cos, sin, c["layout"]))
    return s["Kc"], s["Vc"], s["Qo"]


def _plain_attention(s):
    c = s["case"]
    T, Hq, D = s["Q"].shape
    Hkv, B, P = c["Hkv"], c["B"], c["prefix"]
    g = Hq // Hkv
    L = s["max_len"]
    pages = s["table"].clamp(min=0).long()
    K = s["Kc"][pages].flatten(1, 2)[:, :L].float()
    V = s["Vc"][pages].flatten(1, 2)[:, :L].float()
    i = torch.arange(s["max_q"], device="cuda")[None, :]
    q_len = (s["cu"][1:] - s["cu"][:-1])[:, None]
    tok = torch.where(i < q_len, s["cu"][:-1, None] + i, T).long()
    Q = s["Q"][tok.clamp(max=T - 1)].float().unflatten(2, (Hkv, g)) * D ** -0.5
    S = torch.einsum("bqhgd,blhd->bhgql", Q, K)
    last = s["lens"][:, None] - q_len + i
    seen = torch.arange(L, device="cuda") <= last[:, None, None, :, None]
    S = torch.where(seen, S, float("-inf"))
    if P:
        Kp = s["Kc"][s["prefix_table"].long()].flatten(0, 1)[:P].float()
        Vp = s["Vc"][s["prefix_table"].long()].flatten(0, 1)[:P].float()
        S = torch.cat([torch.einsum("bqhgd,lhd->bhgql", Q, Kp), S], -1)
    m = S.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    p = torch.exp(S - m)
    l = p.sum(-1, keepdim=True)
    O = torch.einsum("bhgql,blhd->bhgqd", p[..., P:], V)
    if P:
        O = O + torch.einsum("bhgql,lhd->bhgqd", p[..., :P], Vp)
    O = torch.where(l > 0, O / l, 0.0)
    lse = (m + torch.log(l)).squeeze(-1)
    # rows of the padded batch that no token has fall behind the last one
    out = torch.empty(T + 1, Hq, D, device="cuda", dtype=s["Q"].dtype)
    out[tok] = O.permute(0, 3, 1, 2, 4).flatten(2, 3).to(out.dtype)
    out_lse = torch.empty(T + 1, Hq, device="cuda")
    out_lse[tok] = lse.permute(0, 3, 1, 2).flatten(2, 3)
    return out[:T], out_lse[:T]


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["op"] == "rope":
        cos, sin = _angles(state["pos"], state["freqs"], state["sections"])
        cos, sin = cos[:, None], sin[:, None]
        sin = -sin if c["inverse"] else sin
        return (_rotate(state["Q"], cos, sin, c["layout"]),
                _rotate(state["K"], cos, sin, c["layout"]))
    if c["op"] == "append":
        return _plain_append(state)
    return _plain_attention(state)


# ---- what a pass cannot do without --------------------------------------------------------
def work(case):
    e = _SIZE[case["dtype"]]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["op"] == "rope":
        tokens = case["B"] * case["S"]
        values = tokens * (Hq + Hkv) * D
        turned = tokens * (Hq + Hkv) * case["rot"]
        return {"bytes": 2 * e * values + 4 * case["axes"] * tokens, "flops": 3 * turned}
    q, n = _lengths(case)
    T = sum(q)
    if case["op"] == "append":
        return {"bytes": 2 * e * T * (Hq + 2 * Hkv) * D + 8 * T,
                "flops": 3 * T * (Hq + Hkv) * case["rot"]}
    P = case["prefix"]
    keys = sum(n) + P
    seen = sum(qi * ni - qi * (qi - 1) // 2 for qi, ni in zip(q, n)) + T * P
    return {"bytes": 2 * e * keys * Hkv * D + 2 * e * T * Hq * D + 4 * T * Hq,
            "flops": 4 * seen * Hq * D}


# ---- the definitions in 64 bits -----------------------------------------------------------
def _turn64(x, pos, freqs, sections, layout, sign):
    """x [tokens, heads, D] turned by pos [axes, tokens], as complex numbers."""
    half = freqs.numel()
    start, parts = 0, []
    for a, width in enumerate(sections):
        parts.append(pos[a].double()[:, None] * freqs[None, start:start + width])
        start += width
    w = torch.polar(torch.ones(1, dtype=torch.float64, device=x.device),
                    sign * torch.cat(parts, 1))[:, None, :]
    y = x.double().clone()
    if layout == "halves":
        first, second = slice(0, half), slice(half, 2 * half)
    else:
        first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
    z = torch.complex(y[..., first], y[..., second]) * w
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        outs = []
        for x in (s["Q"], s["K"]):
            per = []
            for b in range(case["B"]):
                y = _turn64(x[b].transpose(0, 1), s["pos"][:, b], s["freqs"], s["sections"],
                            case["layout"], -1.0 if case["inverse"] else 1.0)
                per.append(y.transpose(0, 1))
            outs.append(torch.stack(per))
        return tuple(outs)
    q, n = _lengths(case)
    page, Hq, Hkv = case["page"], case["Hq"], case["Hkv"]
    g = Hq // Hkv
    if case["op"] == "append":
        Kc, Vc, Qo = s["Kc"].double(), s["Vc"].double(), s["Q"].double()
        t = 0
        for b in range(case["B"]):
            rows = slice(t, t + q[b])
            place = torch.arange(n[b] - q[b], n[b], device="cuda")
            pos = place[None] if s["pos"] is None else s["pos"][:, rows]
            where = s["table"][b].long()[place // page] * page + place % page
            turned = _turn64(s["K"][rows], pos, s["freqs"], s["sections"], case["layout"], 1.0)
            Kc.view(-1, *Kc.shape[2:])[where] = turned
            Vc.view(-1, *Vc.shape[2:])[where] = s["V"][rows].double()
            Qo[rows] = _turn64(s["Q"][rows], pos, s["freqs"], s["sections"], case["layout"], 1.0)
            t += q[b]
        return Kc, Vc, Qo
    P, D = case["prefix"], case["D"]
    O = torch.zeros(sum(q), Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(sum(q), Hq, dtype=torch.float64, device="cuda")
    flatK, flatV = (s[k].reshape(-1, Hkv, D) for k in ("Kc", "Vc"))
    ahead = torch.arange(P, device="cuda")
    ahead = s["prefix_table"].long()[ahead // page] * page + ahead % page if P else ahead
    t = 0
    for b in range(case["B"]):
        place = torch.arange(n[b], device="cuda")
        where = torch.cat([ahead, s["table"][b].long()[place // page] * page + place % page])
        limit = P + n[b] - q[b] + torch.arange(q[b], device="cuda")
        hidden = torch.arange(P + n[b], device="cuda")[None, :] > limit[:, None]
        for h in range(Hkv):
            k, v = flatK[where, h].double(), flatV[where, h].double()
            x = s["Q"][t:t + q[b], h * g:(h + 1) * g].double().transpose(0, 1)
            z = (x @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
            lse[t:t + q[b], h * g:(h + 1) * g] = torch.logsumexp(z, -1).T
            O[t:t + q[b], h * g:(h + 1) * g] = (torch.softmax(z, -1) @ v).transpose(0, 1)
        t += q[b]
    return O, lse
