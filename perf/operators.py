"""Head norms with rotation, and attention under masks, as cases that can be timed and compared.

A case is a dict of plain values; its "op" says which entry point it goes through:

  norm   ops.head_norm_rope: RMSNorm of every q and k head and the rotation, in one pass
  attn   ops.masked_attn: grouped-head attention with score cap, distance bias, documents,
         prefixes and lengths

Sizes: the token grids of Wan2.2-TI2V-5B (24 heads of 128, 374 tokens a frame, 1080 and 7854
tokens a clip, 512 text tokens), and generic ones (grouped heads 32 over 8, powers of two, odd
lengths).  Lists of numbers are texts: "470,123".
"""
import math

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one generated token of 8 requests at different places: latency
        {"name": "norm_step", "op": "norm", "batch": 8, "len": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "pairs": 64, "halves": True, "table": 8192, "positions": True},
        # a chunk of a prompt of odd length, small heads, half of their channels turned
        {"name": "norm_chunk_f16", "op": "norm", "batch": 3, "len": 517, "heads": 16, "kv_heads": 4, "dim": 64,
         "dtype": "f16", "pairs": 16, "halves": True, "table": 4096, "positions": True},
        # two 368x480x21 clips packed in one row of tokens, each with its own grid positions
        {"name": "norm_packed", "op": "norm", "batch": 1, "len": 2160, "heads": 24, "kv_heads": 24, "dim": 128,
         "dtype": "bf16", "pairs": 64, "halves": False, "table": 1080, "positions": True},
        # the q and k of a 704x544x81 generation with guidance
        {"name": "norm_L7854", "op": "norm", "batch": 2, "len": 7854, "heads": 24, "kv_heads": 24, "dim": 128,
         "dtype": "bf16", "pairs": 64, "halves": False, "table": 7854, "positions": False},
        # one generated token of one request: latency
        {"name": "step_B1", "op": "attn", "batch": 1, "len_q": 1, "len_k": 1000, "heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "causal": True, "cap": 0.0, "reach": 0, "docs": "", "prefix": "", "lens": ""},
        # one generated token of 16 requests over a long cache, every one of another length
        {"name": "step_B16", "op": "attn", "batch": 16, "len_q": 1, "len_k": 8192, "heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "causal": True, "cap": 0.0, "reach": 0, "docs": "", "prefix": "",
         "lens": "8192,8191,7854,7000,6144,8000,5117,4096,8192,7777,6500,7201,3001,8100,6999,1080"},
        # a text encoder over two padded prompts: 512 positions, bias by distance, no scale
        {"name": "text_bias", "op": "attn", "batch": 2, "len_q": 512, "len_k": 512, "heads": 64, "kv_heads": 64,
         "dim": 64, "dtype": "bf16", "causal": False, "cap": 0.0, "reach": 128, "docs": "", "prefix": "",
         "lens": "470,123"},
        # prompts read in full, their continuations causally, odd lengths
        {"name": "prefix_f16", "op": "attn", "batch": 2, "len_q": 2049, "len_k": 2049, "heads": 16, "kv_heads": 4,
         "dim": 64, "dtype": "f16", "causal": True, "cap": 0.0, "reach": 0, "docs": "", "prefix": "512,301", "lens": ""},
        # capped scores over a prompt
        {"name": "cap_L4096", "op": "attn", "batch": 1, "len_q": 4096, "len_k": 4096, "heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "f16", "causal": True, "cap": 50.0, "reach": 0, "docs": "", "prefix": "", "lens": ""},
        # clips of different size packed in one row of tokens, each attending to itself
        {"name": "packed_clips", "op": "attn", "batch": 1, "len_q": 7854, "len_k": 7854, "heads": 24, "kv_heads": 24,
         "dim": 128, "dtype": "bf16", "causal": False, "cap": 0.0, "reach": 0, "docs": "0,374,1454,3698", "prefix": "",
         "lens": ""},
        # the next chunk of a prompt behind a long cache
        {"name": "chunk_16k", "op": "attn", "batch": 2, "len_q": 256, "len_k": 16384, "heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "causal": True, "cap": 0.0, "reach": 0, "docs": "", "prefix": "", "lens": ""},
        # a long prompt
        {"name": "causal_L8192", "op": "attn", "batch": 1, "len_q": 8192, "len_k": 8192, "heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "causal": True, "cap": 0.0, "reach": 0, "docs": "", "prefix": "", "lens": ""},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _numbers(text):
    return [int(t) for t in text.split(",")] if text else []


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def draw(rng):
    if rng.random() < 0.35:
        while True:
            dim = rng.choice([64, 128, 128, 256])
            kv = rng.choice([1, 4, 8, 24])
            case = {"op": "norm", "batch": rng.choice([1, 2, 3, 8]), "len": _log(rng, 1, 8192),
                    "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "dim": dim,
                    "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "pairs": rng.choice([dim // 4, dim // 2, dim // 2]),
                    "halves": rng.random() < 0.5, "table": 0, "positions": rng.random() < 0.5}
            case["table"] = case["len"] + rng.randint(0, 1000)
            if work(case)["bytes"] <= work(listed()[3])["bytes"]:
                return case
    while True:
        kv = rng.choice([1, 4, 8, 24])
        case = {"op": "attn", "batch": rng.choice([1, 1, 2, 3, 16]), "len_q": 0, "len_k": _log(rng, 60, 16384),
                "heads": kv * rng.choice([1, 1, 2, 4, 8]), "kv_heads": kv, "dim": rng.choice([64, 128, 128]),
                "dtype": rng.choice(["bf16", "bf16", "f16"]), "causal": rng.random() < 0.6,
                "cap": rng.choice([0.0, 0.0, 0.0, 20.0, 50.0]), "reach": 0, "docs": "", "prefix": "", "lens": ""}
        n = case["len_k"]
        case["len_q"] = rng.choice([1, n, n, _log(rng, 1, n)])
        if rng.random() < 0.3:
            case["reach"] = _log(rng, 1, 512)
        if case["len_q"] > 1 and rng.random() < 0.4:
            case["docs"] = _text([0] + sorted(rng.sample(range(1, n), rng.randint(1, 6))))
        if case["causal"] and rng.random() < 0.3:
            parts = len(_numbers(case["docs"])) if case["docs"] else case["batch"]
            case["prefix"] = _text(rng.randint(0, max(1, n // 2)) for _ in range(parts))
        if rng.random() < 0.5 and not case["docs"]:
            case["lens"] = _text(rng.randint(max(1, n // 4), n) for _ in range(case["batch"]))
        dense = case["batch"] * case["heads"] * case["len_q"] * n * case["dim"]
        most = listed()[-1]
        if dense <= most["heads"] * most["len_q"] * most["len_k"] * most["dim"] and \
                case["batch"] * case["kv_heads"] * n * case["dim"] <= 16 * 8 * 8192 * 128:
            return case


# ─── inputs, from the seed alone ──────────────────────────────────────────────

def _starts(case):
    """Position of the first query among the keys, per sample: whole sequences begin at 0, chunks and
    single tokens are the last of their sample."""
    lens = _numbers(case["lens"]) or [case["len_k"]] * case["batch"]
    whole = case["len_q"] == case["len_k"]
    return lens, [0 if whole else n - case["len_q"] for n in lens]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    def ints(values, *shape):
        return torch.tensor(values, dtype=torch.int32, device="cuda").reshape(shape)

    B, D = case["batch"], case["dim"]
    if case["op"] == "norm":
        L, width = case["len"], (case["heads"] + case["kv_heads"]) * D
        # q and k are views of one projection's output, its channels of different size
        x = (normal(B, L, width) * (0.5 + normal(width).abs())).to(dt)
        q, k = x.split([case["heads"] * D, case["kv_heads"] * D], dim=-1)
        angle = torch.rand(case["table"], case["pairs"], generator=g, device="cuda") * (2 * math.pi)
        pos = None
        if case["positions"]:
            pos = torch.randint(0, case["table"], (B, L), generator=g, device="cuda", dtype=torch.int32)
        return {"case": case, "q": q.unflatten(-1, (-1, D)), "k": k.unflatten(-1, (-1, D)),
                "gamma_q": (1 + 0.5 * normal(D).abs()).to(dt), "gamma_k": (1 + 0.5 * normal(D).abs()).to(dt),
                "cos": angle.cos(), "sin": angle.sin(), "positions": pos}
    # normed heads; a model without a scale keeps its queries small instead
    H, Hk, R = case["heads"], case["kv_heads"], case["reach"]
    scale = 1.0 if R else D ** -0.5
    q = (normal(B, case["len_q"], H, D) * (D ** -0.5 / scale)).to(dt)
    k, v = (normal(B, case["len_k"], Hk, D).to(dt) for _ in range(2))
    lens, starts = _starts(case)
    docs, prefix = _numbers(case["docs"]), _numbers(case["prefix"])
    bias = None
    if R:    # falls off with distance, each head at its own rate, uneven as trained tables are
        far = (torch.arange(2 * R + 1, device="cuda") - R).abs()
        bias = normal(H, 2 * R + 1) * 0.5 - normal(H, 1).abs() * torch.log1p(far.float())
    return {"case": case, "q": q, "k": k, "v": v, "scale": scale, "bias": bias,
            "doc_starts": ints(docs * B, B, len(docs)) if docs else None,
            "prefix_lens": (ints(prefix * B, B, len(docs)) if docs else ints(prefix, B)) if prefix else None,
            "seqlen_k": ints(lens, B) if case["lens"] else None,
            "q_start": ints(starts, B) if case["lens"] else None}


# ─── one pass ─────────────────────────────────────────────────────────────────

_package = None


def _ops():
    global _package
    if _package is None:
        import __graft_entry__
        _package = __graft_entry__.load_package()
    return _package.ops


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        if own:
            return _ops().head_norm_rope(state["q"], state["k"], state["gamma_q"], state["gamma_k"], EPS, state["cos"],
                                         state["sin"], state["positions"], not case["halves"])
        return tuple(_plain_norm(state[x], state["gamma_" + x], state) for x in "qk")
    if own:
        return _ops().masked_attn(state["q"], state["k"], state["v"], state["scale"], case["causal"], case["cap"],
                                  state["bias"], state["doc_starts"], state["prefix_lens"], state["seqlen_k"],
                                  state["q_start"])
    return _plain_attn(state)


def _plain_norm(x, gamma, state):
    P, halves = state["case"]["pairs"], state["case"]["halves"]
    f = x.float()
    f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * gamma.float()
    if state["positions"] is None:
        c, s = (state[t][:x.shape[1]][None, :, None] for t in ("cos", "sin"))
    else:
        c, s = (state[t][state["positions"].long()][:, :, None] for t in ("cos", "sin"))
    turned, rest = f[..., :2 * P], f[..., 2 * P:]
    if halves:
        a, b = turned[..., :P], turned[..., P:]
        turned = torch.cat((a * c - b * s, a * s + b * c), -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    return torch.cat((turned, rest), -1).to(x.dtype)


# scores held at once by the plain form
_SCORES = 1 << 28


def _plain_attn(state):
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    G, R, cap = H // Hk, case["reach"], case["cap"]
    j = torch.arange(Lk, device=q.device)
    out = torch.empty_like(q)
    rows = max(1, _SCORES // (H * Lk))
    for b in range(B):
        kb, vb = (t[b].float().transpose(0, 1).contiguous() for t in (k, v))            # [Hk, Lk, D]
        kt = kb.transpose(1, 2).contiguous()
        start = Lk - Lq if state["q_start"] is None else state["q_start"][b]
        doc_j = None
        if state["doc_starts"] is not None:
            doc_j = torch.searchsorted(state["doc_starts"][b].long(), j, right=True)
        for i0 in range(0, Lq, rows):
            qi = q[b, i0:i0 + rows].float()
            n = qi.shape[0]
            s = qi.view(n, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * n, D) @ kt * state["scale"]
            s = s.view(H, n, Lk)
            if cap:
                s = cap * torch.tanh(s / cap)
            p = torch.arange(i0, i0 + n, device=q.device) + start
            if R:
                s = s + state["bias"][:, (j[None] - p[:, None]).clamp(-R, R) + R]
            see = torch.ones(n, Lk, dtype=torch.bool, device=q.device)
            if doc_j is not None:
                doc_p = torch.searchsorted(state["doc_starts"][b].long(), p, right=True)
                see &= (doc_j[None] == doc_p[:, None]) & (doc_p[:, None] > 0)
            if case["causal"]:
                past = j[None] <= p[:, None]
                if state["prefix_lens"] is not None:
                    first, length = 0, state["prefix_lens"][b].long()
                    if doc_j is not None:
                        at = (doc_p - 1).clamp(min=0)
                        first, length = state["doc_starts"][b].long()[at][:, None], length[at][:, None]
                    past = past | (j[None] < first + length)
                see &= past
            if state["seqlen_k"] is not None:
                see &= j[None] < state["seqlen_k"][b]
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
            e = torch.exp(s - top)
            total = e.sum(-1, keepdim=True)
            e = e / torch.where(total == 0, torch.ones_like(total), total)
            o = (e.view(Hk, G * n, Lk) @ vb).view(Hk, G, n, D)
            out[b, i0:i0 + n] = o.permute(2, 0, 1, 3).reshape(n, H, D).to(q.dtype)
    return out


# ─── what a pass cannot do without ────────────────────────────────────────────

def _intervals(case):
    """(sample, keys that each of its query rows sees as (first, end)) on the host."""
    lens, starts = _starts(case)
    docs, prefix = _numbers(case["docs"]), _numbers(case["prefix"])
    for b in range(case["batch"]):
        rows = []
        for i in range(case["len_q"]):
            p = starts[b] + i
            lo, hi, length = 0, lens[b], prefix[b] if prefix and not docs else 0
            if docs:
                at = sum(d <= p for d in docs) - 1
                if at < 0:
                    rows.append((0, 0))
                    continue
                lo = docs[at]
                hi = min(hi, docs[at + 1] if at + 1 < len(docs) else case["len_k"])
                length = prefix[at] if prefix else 0
            if case["causal"]:
                hi = min(hi, max(p + 1, lo + length))
            rows.append((lo, max(lo, hi)))
        yield b, rows


def work(case):
    size = TYPES[case["dtype"]].itemsize
    D = case["dim"]
    if case["op"] == "norm":
        values = case["batch"] * case["len"] * (case["heads"] + case["kv_heads"]) * D
        rows = min(case["table"], case["batch"] * case["len"]) if case["positions"] else case["len"]
        pos = 4 * case["batch"] * case["len"] if case["positions"] else 0
        return {"bytes": 2 * values * size + rows * case["pairs"] * 8 + 2 * D * size + pos, "flops": 10 * values}
    pairs = keys = 0
    for _, rows in _intervals(case):
        pairs += sum(hi - lo for lo, hi in rows)
        ends, seen = 0, 0            # keys that any row sees (first keys and ends only grow along the rows)
        for lo, hi in rows:
            seen += max(0, hi - max(lo, ends))
            ends = max(ends, hi)
        keys += seen
    moved = 2 * case["batch"] * case["len_q"] * case["heads"] * D + 2 * keys * case["kv_heads"] * D
    return {"bytes": moved * size + case["heads"] * (2 * case["reach"] + 1) * 4 * bool(case["reach"]),
            "flops": 4 * D * case["heads"] * pairs}


# ─── the definition in 64 bits ────────────────────────────────────────────────

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        outs = []
        for name in "qk":
            x, P = state[name].double(), case["pairs"]
            y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * state["gamma_" + name].double()
            at = torch.arange(x.shape[1], device=x.device).expand(x.shape[:2]) if state["positions"] is None \
                else state["positions"].long()
            turn = torch.complex(state["cos"].double(), state["sin"].double())[at].unsqueeze(2)
            first, second = (slice(0, P), slice(P, 2 * P)) if case["halves"] else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
            z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
            y[..., first], y[..., second] = z.real, z.imag
            outs.append(y)
        return tuple(outs)
    q, k, v = (state[t].double() for t in "qkv")
    G = case["heads"] // case["kv_heads"]
    lens, starts = _starts(case)
    out = torch.zeros_like(q)
    rows = max(1, (1 << 27) // case["len_k"])
    for b, seen in _intervals(case):
        lo, hi = (torch.tensor([r[e] for r in seen], device=q.device) for e in (0, 1))
        for h in range(case["heads"]):
            kh, vh = k[b, :, h // G].t().contiguous(), v[b, :, h // G].contiguous()
            for i0 in range(0, case["len_q"], rows):
                i1 = min(case["len_q"], i0 + rows)
                # of these rows, the keys that any of them sees
                first, end = int(lo[i0:i1].min()), int(hi[i0:i1].max())
                if end <= first:
                    continue
                at = torch.arange(first, end, device=q.device)
                s = torch.mm(q[b, i0:i1, h], kh[:, first:end].contiguous()) * state["scale"]
                if case["cap"]:
                    s = (s / case["cap"]).tanh() * case["cap"]
                if case["reach"]:
                    off = at[None] - (torch.arange(i0, i1, device=q.device)[:, None] + starts[b])
                    s = s + state["bias"][h].double()[off.clamp(-case["reach"], case["reach"]) + case["reach"]]
                hidden = (at[None] < lo[i0:i1, None]) | (at[None] >= hi[i0:i1, None])
                w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
                out[b, i0:i1, h] = torch.mm(w.masked_fill(hidden, 0.0).nan_to_num(0.0), vh[first:end])
    return out
