"""ops.masked_attn: attention with capped scores, a bias by distance, documents, prefixes, lengths and
grouped heads, against the definition in 64 bits; its refusals on the CPU."""
import ctypes
import math

import pytest
import torch

DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16
STEP = {BF: 2 ** -8, HF: 2 ** -11}
LOWEST = torch.finfo(torch.float32).min


# ─── on the CPU ───────────────────────────────────────────────────────────────

def test_abi_refusals(W):
    N = W._native
    lib = N.lib()
    P = 256         # an aligned stand-in address: every call fails before a launch
    t = N.WanTensor(P, 4096, 512, 64)

    def call(q=t, k=t, v=t, out=t, B=1, Hq=4, Hk=2, Lq=8, Lk=8, D=64, dtype=0, scale=0.1, ws=None, n=0, **mask):
        m = N.WanAttnMask(**mask)
        rc = lib.wan_masked_attn(q, k, v, out, B, Hq, Hk, Lq, Lk, D, dtype, scale, ctypes.byref(m), ws, n, None)
        return rc, N.last_error() if rc else ""

    null = N.WanTensor(0, 0, 0, 0)
    for kw, code, what in ((dict(scale=0.0), 2, "softmax_scale"), (dict(scale=float("inf")), 2, "softmax_scale"),
                           (dict(B=-1), 1, "negative"), (dict(D=96), 2, "head_dim"), (dict(dtype=2), 2, "dtype"),
                           (dict(Hk=3), 1, "multiple"), (dict(Hk=0), 1, "multiple"), (dict(Lk=(1 << 30) + 1), 2, "2^30"),
                           (dict(Lq=1 << 30), 2, "2^30"), (dict(q=null), 1, "NULL"), (dict(v=null), 1, "NULL"),
                           (dict(out=null), 1, "NULL"), (dict(k=N.WanTensor(P + 8, 4096, 512, 64)), 1, "aligned"),
                           (dict(k=N.WanTensor(P, 4096, 516, 64)), 1, "stride"),
                           (dict(k=N.WanTensor(P, 4096, -512, 64)), 1, "negative"),
                           (dict(v=N.WanTensor(P, 4096, 1 << 24, 64)), 2, "token stride"),
                           (dict(softcap=-1.0), 1, "softcap"), (dict(softcap=float("nan")), 1, "softcap"),
                           (dict(softcap=1e31), 1, "softcap"), (dict(softcap=float("inf")), 1, "softcap"),
                           (dict(Lq=(1 << 29) + 1), 2, "2^29"),
                           (dict(bias=P, bias_reach=-1), 1, "bias_reach"), (dict(doc_starts=P), 1, "docs"),
                           (dict(prefix_lens=P), 1, "prefix_lens"), (dict(seqlen_k=P + 2), 1, "aligned"),
                           (dict(ws=P + 16, n=1 << 20), 1, "workspace")):
        rc, msg = call(**kw)
        assert rc == code and what in msg and msg.startswith("wan_masked_attn"), (kw, rc, msg)
    assert call(B=0)[0] == call(Hq=0)[0] == call(Lq=0)[0] == 0


def test_operator_refuses_host_tensors_and_traces(W):
    x = torch.zeros(1, 4, 2, 64, dtype=BF)
    with pytest.raises(ValueError, match="CUDA"):
        W.ops.masked_attn(x, x, x, 0.1)
    q, k = torch.empty(2, 5, 6, 64, device="meta", dtype=BF), torch.empty(2, 9, 3, 64, device="meta", dtype=BF)
    assert torch.ops.wan_hip.masked_attn(q, k, k, 0.1, True).shape == q.shape


# ─── the definition in 64 bits ────────────────────────────────────────────────

def _see(B, Lq, Lk, causal, docs, prefix, lens, starts):
    """[B, Lq, Lk] truth values, pair by pair."""
    j = torch.arange(Lk)
    out = torch.zeros(B, Lq, Lk, dtype=torch.bool)
    for b in range(B):
        p = (Lk - Lq if starts is None else int(starts[b])) + torch.arange(Lq)
        see = (j < (Lk if lens is None else int(lens[b])))[None].expand(Lq, Lk).clone()
        at = None
        if docs is not None:
            d = docs[b].long()
            at_j, at = torch.bucketize(j, d, right=True), torch.bucketize(p, d, right=True)
            see &= (at_j[None] == at[:, None]) & (at[:, None] > 0)
        if causal:
            ok = j[None] <= p[:, None]
            if prefix is not None:
                if docs is None:
                    ok |= (j < int(prefix[b]))[None]
                else:
                    k = (at - 1).clamp(min=0)
                    ok |= j[None] < (docs[b].long()[k] + prefix[b].long()[k])[:, None]
            see &= ok
        out[b] = see
    return out


def _reference(q, k, v, scale, causal=False, cap=0.0, bias=None, docs=None, prefix=None, lens=None, starts=None):
    """(out, allowed error) by the definition in 64 bits.

    The error: a weight is rounded to the type (u of it), and the sum that divides takes the rounded ones;
    the output is rounded (u).  Scores in fp32: D products and sums of 2^-24 each of sum |q k|, then a handful
    of operations on a value of up to |s| + |bias| + cap, the tanh 2^-22 of the cap; a weight is off by the
    score's error (times 2: against the reference point), its exponential and the rescalings by 2^-20; the
    sums over n keys by n 2^-24.  fp16 weights below 2^-14 of the largest are off by 2^-25 of it."""
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    see = _see(B, Lq, Lk, causal, *(t if t is None else t.cpu() for t in (docs, prefix, lens, starts))).to(q.device)
    u = STEP[q.dtype]
    out, tol = torch.zeros(B, Lq, H, D, dtype=torch.float64, device=q.device), torch.zeros(B, Lq, H, D, dtype=torch.float64,
                                                                                          device=q.device)
    for b in range(B):
        p = (Lk - Lq if starts is None else int(starts[b])) + torch.arange(Lq, device=q.device)
        for h in range(H):
            qh, kh, vh = q[b, :, h].double(), k[b, :, h // (H // Hk)].double(), v[b, :, h // (H // Hk)].double()
            s = torch.mm(qh, kh.t().contiguous()) * scale
            es = torch.mm(qh.abs(), kh.abs().t().contiguous()) * scale * ((D + 4) * 2 ** -24)
            es = es + (s.abs() if not cap else s.abs().clamp(max=cap)) * 2 ** -21
            if cap:
                s = cap * torch.tanh(s / cap)
                es = es + cap * 2 ** -22
            if bias is not None:
                R = bias.shape[1] // 2
                add = bias[h].double()[(torch.arange(Lk, device=q.device)[None] - p[:, None]).clamp(-R, R) + R]
                s = s + add
                es = es + add.abs().clamp(max=1e30) * 2 ** -22
            s = s.masked_fill(~see[b], -math.inf)
            es = es.masked_fill(~see[b] | s.isinf(), 0)
            w = torch.softmax(s, -1)
            w = w.masked_fill((s == -math.inf).all(-1, keepdim=True) | ~see[b], 0.0)
            vv = vh.masked_fill(~see[b].any(0)[:, None], 0.0)
            o = torch.mm(w, vv)
            size = torch.mm(w, vv.abs())
            weight_off = u + 2 * (w * es).sum(-1, keepdim=True) + 2 ** -20 + Lk * 2 ** -23
            out[b, :, h] = o
            # numerator term by term, then the common divisor
            tol[b, :, h] = torch.mm(w * (u + 2 * es + 2 ** -20 + Lk * 2 ** -23), vv.abs()) + weight_off * o.abs() + \
                u * o.abs() + 2 ** -24 * size
            if q.dtype == HF:
                tol[b, :, h] += Lk * 2 ** -25 * w.amax(-1, keepdim=True) * vv.abs().amax() + 2 ** -25
    return out, tol * (1 + 2 ** -6)


def _make(B, Lq, Lk, Hq, Hk, D, dtype, seed, reach=None, spread=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=g, device=DEV)
    q = (normal(B, Lq, Hq, D) * spread).to(dtype)
    k, v = (normal(B, Lk, Hk, D).to(dtype) for _ in range(2))
    bias = None if reach is None else normal(Hq, 2 * reach + 1) * 2
    return q, k, v, bias


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _check(W, q, k, v, scale, **kw):
    names = {"cap": "softcap", "docs": "doc_starts", "prefix": "prefix_lens", "lens": "seqlen_k", "starts": "q_start"}
    got = W.ops.masked_attn(q, k, v, scale, **{names.get(n, n): x for n, x in kw.items()})
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    want, tol = _reference(q, k, v, scale, **kw)
    off = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all()
    bad = off > tol
    assert not bad.any(), (int(bad.sum()), float((off / tol.clamp(min=1e-300)).max()), bad.nonzero()[:4].tolist())
    return got


# queries, keys, query heads, k/v heads
SIZES = [(1, 1, 1, 1), (1, 33, 8, 1), (1, 1000, 32, 8), (2, 31, 3, 3), (5, 64, 6, 2), (33, 65, 40, 1), (37, 37, 4, 4),
         (64, 200, 4, 2), (129, 129, 2, 1), (255, 257, 2, 2), (257, 511, 3, 1), (300, 1100, 8, 4), (700, 700, 2, 2),
         (520, 520, 16, 2), (1030, 1030, 1, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Lq,Lk,Hq,Hk", SIZES)
def test_sizes(W, Lq, Lk, Hq, Hk, causal, D, dtype):
    q, k, v, _ = _make(2, Lq, Lk, Hq, Hk, D, dtype, Lq + Lk)
    _check(W, q, k, v, D ** -0.5, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("cap", [0.5, 20.0, 50.0, 256.0, 257.0, 1e6])
@pytest.mark.parametrize("Lq,Lk,Hq,Hk", [(1, 300, 8, 2), (200, 333, 4, 2), (600, 600, 2, 1)])
def test_cap(W, Lq, Lk, Hq, Hk, cap, dtype, D):
    q, k, v, _ = _make(1, Lq, Lk, Hq, Hk, D, dtype, 7, spread=3.0)
    _check(W, q, k, v, 2 * D ** -0.5, causal=True, cap=cap)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("cap", [1e9, 1e30])
@pytest.mark.parametrize("Lq,Lk", [(1, 300), (300, 333)])
def test_caps_beyond_every_score_change_nothing(W, Lq, Lk, cap, dtype, D):
    """With |s| < 2^10 the cap takes s (s / cap)^2 / 3 < 2^-29 of a score: the uncapped result, to its rounding."""
    q, k, v, _ = _make(1, Lq, Lk, 4, 2, D, dtype, 8, spread=3.0)
    want, tol = _reference(q, k, v, 2 * D ** -0.5)
    assert ((W.ops.masked_attn(q, k, v, 2 * D ** -0.5, softcap=cap).double() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e-38, 1e-30, 1e-6])
@pytest.mark.parametrize("Lq,Lk", [(1, 300), (300, 333)])
def test_caps_far_below_the_scores(W, Lq, Lk, cap):
    q, k, v, _ = _make(1, Lq, Lk, 4, 2, 128, BF, 9, spread=3.0)
    q[:, :, 0] = 0
    _check(W, q, k, v, 2 * 128 ** -0.5, cap=cap)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128)])
@pytest.mark.parametrize("reach", [0, 1, 31, 128, 4000])
@pytest.mark.parametrize("Lq,Lk,Hq,Hk,causal,cap", [(1, 300, 8, 2, True, 0.0), (512, 512, 4, 4, False, 0.0),
                                                    (200, 1333, 32, 1, False, 0.0), (37, 2600, 1, 1, True, 30.0),
                                                    (900, 901, 40, 4, True, 0.0), (1, 2500, 64, 1, False, 0.0)])
def test_bias(W, Lq, Lk, Hq, Hk, causal, cap, reach, dtype, D):
    q, k, v, bias = _make(1, Lq, Lk, Hq, Hk, D, dtype, reach, reach, spread=0.3)
    _check(W, q, k, v, 1.0, causal=causal, cap=cap, bias=bias)


@pytest.mark.gpu
def test_bias_that_spans_the_windows(W):
    """Tables and keys far larger than what a block holds of them."""
    q, k, v, bias = _make(1, 3, 20000, 2, 1, 64, BF, 5, 19000)
    _check(W, q, k, v, 0.125, bias=bias)
    q, k, v, bias = _make(1, 9000, 9000, 1, 1, 64, BF, 6, 8000)
    _check(W, q, k, v, 0.125, bias=bias, causal=True)


DOCS = [[[0, 5, 90, 130]], [[0, 64, 128, 256]], [[3, 10, 33, 299]], [[0, 0, 70, 70]], [[0, 100, 1000, 2000]], [[150, 151, 152, 153]]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("docs", DOCS)
@pytest.mark.parametrize("causal,prefix", [(False, None), (True, None), (True, [[2, 40, 0, 500]])])
@pytest.mark.parametrize("Lq,Lk,Hq,Hk", [(300, 300, 2, 2), (40, 300, 8, 2)])
def test_documents(W, Lq, Lk, Hq, Hk, docs, causal, prefix, dtype, D):
    q, k, v, _ = _make(2, Lq, Lk, Hq, Hk, D, dtype, 3)
    second = [[0, 20, 40, 60]]
    _check(W, q, k, v, D ** -0.5, causal=causal, docs=_ints(docs + second),
           prefix=None if prefix is None else _ints(prefix + [[1, 0, 20, 21]]))


MANY = {"large": [0, 700, 701, 1500, 1560, 2300], "one_large": [0, 20, 40, 2400], "late": [900, 1000, 2999], "even": list(range(0, 3000, 30)),
        "odd": [0] + [7 + 13 * i + (i % 5) * 2 for i in range(200)], "outside": [-50, 0, 1200, 3000, 3500], "same": [0, 5, 5, 5, 1400, 1400]}


@pytest.mark.gpu
@pytest.mark.parametrize("D,causal", [(64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("which", list(MANY))
@pytest.mark.parametrize("Lq,Hq,Hk", [(3000, 2, 1), (1800, 1, 1), (7, 4, 2), (1, 3, 1)])
def test_many_documents(W, Lq, Hq, Hk, which, D, causal):
    """Blocks of rows that begin with the large documents and hold runs of small ones; more than 64 documents; starts
    outside the keys; empty documents."""
    q, k, v, bias = _make(2, Lq, 3000, Hq, Hk, D, BF, 6, 60 if which == "odd" else None)
    first = MANY[which]
    other = sorted((37 * i * i + 11 * i) % 3000 for i in range(len(first)))
    _check(W, q, k, v, D ** -0.5, causal=causal, bias=bias, docs=_ints([first, other]))


@pytest.mark.gpu
@pytest.mark.parametrize("starts", [[2500, 100, 50, 1700], [2 ** 31 - 1, 0, -(2 ** 31), 5], [0, 3000, 10, 2000]])
def test_documents_out_of_order_write_every_row_in_bounds(W, starts):
    N, lib = W._native, W._native.lib()
    for D, Lq in ((64, 3000), (128, 2777)):
        q, k, v, _ = _make(1, Lq, 3000, 2, 1, D, BF, 8)
        whole = torch.full((1, Lq + 2, 2, D), float("nan"), device=DEV, dtype=BF)
        out, docs = whole[:, 1:-1], _ints([starts])
        mask = N.WanAttnMask(doc_starts=docs.data_ptr(), docs=4)
        N.check("wan_masked_attn", lib.wan_masked_attn(
            N.tensor4(q), N.tensor4(k), N.tensor4(v), N.tensor4(out), 1, 2, 1, Lq, 3000, D, 0, 0.1, ctypes.byref(mask), None, 0,
            torch.cuda.current_stream().cuda_stream))
        assert torch.isfinite(out.float()).all() and (out.float().abs() <= v.float().abs().max()).all()
        assert whole[:, 0].isnan().all() and whole[:, -1].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [[0, 0], [1, 700], [64, 333], [2 ** 31 - 1, -5]])
@pytest.mark.parametrize("Lq,Lk,Hq,Hk", [(700, 700, 4, 2), (1, 90, 4, 4), (100, 700, 2, 1)])
def test_prefix(W, Lq, Lk, Hq, Hk, prefix):
    q, k, v, _ = _make(2, Lq, Lk, Hq, Hk, 128, BF, 4)
    _check(W, q, k, v, 0.09, causal=True, prefix=_ints(prefix))


@pytest.mark.gpu
@pytest.mark.parametrize("Lq", [1, 5, 32, 300])
def test_prefix_of_a_document_that_began_before_the_keys(W, Lq):
    """The prefix counts from the document's first position, whether or not there is a key."""
    q, k, v, _ = _make(2, Lq, 300, 4, 2, 64, BF, 17)
    _check(W, q, k, v, 0.125, causal=True, docs=_ints([[-40, 90, 200], [-7, -2, 30]]),
           prefix=_ints([[60, 20, 300], [3, 20, 9]]), starts=_ints([0, 300 - Lq]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("lens,starts", [([300, 7, 0], None), ([299, 64, 65], [299, 63, 64]), ([-3, 400, 1], [0, 0, 0]),
                                         ([100, 200, 300], [90, 190, 290]), ([300, 300, 300], [-10, 5000, -(2 ** 31)])])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Lq", [1, 10, 300])
def test_lengths_and_starts(W, Lq, causal, lens, starts, dtype, D):
    q, k, v, bias = _make(3, Lq, 300, 8, 2, D, dtype, 9, 40)
    clamped = None if starts is None else _ints([max(s, -(2 ** 30 - 1)) for s in starts])
    got = W.ops.masked_attn(q, k, v, 0.1, causal, 0.0, bias, None, None, _ints(lens), None if starts is None else _ints(starts))
    want, tol = _reference(q, k, v, 0.1, causal=causal, bias=bias, lens=_ints(lens), starts=clamped)
    assert ((got.double() - want).abs() <= tol).all()
    empty = ~_see(3, Lq, 300, causal, None, None, lens, None if starts is None else clamped.cpu()).any(-1)
    assert (got[empty.to(DEV)] == 0).all() and (empty.any() or causal or min(lens) > 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("Lq,causal,docs,lens", [(1, False, None, 170), (200, True, None, 200), (200, False, [0, 70, 75, 133], 200),
                                                 (600, True, [0, 9, 310], 600), (600, False, None, 431)])
def test_masked_keys_do_not_reach_a_row(W, Lq, causal, docs, lens, value, dtype):
    """Rows that do not see a bad k row are as without it, bit for bit, and as the definition has them with a bad v
    row (their weights may then be rounded at another reference point); rows that see a bad v row get the value,
    or NaN, in its channel alone."""
    Lk = max(Lq, 200)
    q, k, v, _ = _make(1, Lq, Lk, 4, 2, 128, dtype, 11)
    kw = dict(causal=causal, doc_starts=None if docs is None else _ints([docs]), seqlen_k=_ints([lens]))
    good = W.ops.masked_attn(q, k, v, 0.1, **kw)
    want, tol = _reference(q, k, v, 0.1, causal=causal, docs=kw["doc_starts"], lens=kw["seqlen_k"])
    see = _see(1, Lq, Lk, causal, None if docs is None else torch.tensor([docs]), None, [lens], None)[0].to(DEV)
    bad = [j for j in (5, 72, 131, 198, Lk - 1) if j < Lk]
    for which in (k, v):
        old = which.clone()
        for j in bad:
            which[0, j, 1, 3] = value
        got = W.ops.masked_attn(q, k, v, 0.1, **kw)
        hit = see[:, bad].any(-1)
        assert torch.equal(got[0, :, :2], good[0, :, :2])          # the other k/v head's
        if which is k:
            assert torch.equal(got[0, ~hit], good[0, ~hit])
        else:
            poisoned = torch.zeros_like(got[0], dtype=torch.bool)
            poisoned[hit, 2:, 3] = True
            assert not torch.isfinite(got[0][poisoned].float()).any()
            assert ((got[0].double() - want[0]).abs() <= tol[0])[~poisoned].all()
        which.copy_(old)


@pytest.mark.gpu
@pytest.mark.parametrize("Lq", [1, 100, 513])
def test_lowest_and_infinite_bias(W, Lq):
    """The lowest value for some distances, for all (uniform, as softmax has it), and -inf for all (zeros)."""
    q, k, v, bias = _make(1, Lq, 600, 3, 1, 64, BF, 2, 300)
    bias[0, ::3] = LOWEST
    bias[1] = LOWEST
    bias[2] = -math.inf
    got = W.ops.masked_attn(q, k, v, 0.1, bias=bias)
    want, tol = _reference(q, k, v, 0.1, bias=torch.where(bias == LOWEST, -1e30, bias.double()).float())
    assert ((got[:, :, 0].double() - want[:, :, 0]).abs() <= tol[:, :, 0]).all()
    mean = v[0, :, 0].double().mean(0)
    assert ((got[0, :, 1].double() - mean).abs() <= mean.abs() * 2 ** -8 + 600 * 2 ** -23).all()
    assert (got[:, :, 2] == 0).all()
    bias[:, 300:] = -math.inf           # keys at and behind the position are hidden: the first row of all sees none
    full = W.ops.masked_attn(q, k[:, :Lq], v[:, :Lq], 0.1, bias=bias)
    assert (full[0, 0] == 0).all() and torch.isfinite(full.float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [0.0, 40.0])
def test_equal_and_steep_scores(W, spread):
    """All scores 0, and scores of some hundred that grow along the keys (the running max moves at every tile)."""
    for Lq in (1, 300):
        q, k, v, _ = _make(1, Lq, 1000, 2, 1, 64, HF, 8)
        q = torch.full_like(q, spread)
        k = (torch.linspace(-1, 1, 1000, device=DEV)[None, :, None, None] * torch.ones_like(k, dtype=torch.float32)).half()
        _check(W, q, k, v, 0.125)
        _check(W, q, k.flip(1), v, 0.125, causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("Lq", [1, 300])
def test_strides(W, Lq):
    """Head-major caches, views of one projection, a k/v shared by the batch."""
    g = torch.Generator(device=DEV).manual_seed(1)
    cache = torch.randn(2, 2, 4, 333, 136, generator=g, device=DEV).to(BF)
    k, v = (t[:, :, 3:, 8:].transpose(1, 2) for t in cache)
    q = torch.randn(2, Lq, 3 * 8 * 128, generator=g, device=DEV).to(BF)[..., 1024:2048].unflatten(-1, (8, 128))
    _check(W, q, k, v, 0.1, causal=True)
    _check(W, q, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1), 0.1, lens=_ints([330, 12]))


@pytest.mark.gpu
@pytest.mark.parametrize("Lq", [1, 260])
def test_offsets_beyond_32_bits(W, Lq):
    """The last keys of a cache of 2.6e9 values in each of k and v."""
    Lk, H, D = 320000, 64, 128
    k, v = (torch.zeros(1, Lk, H, D, device=DEV, dtype=BF) for _ in range(2))
    q, kt, vt, _ = _make(1, Lq, 1000, H, H, D, BF, 3)
    k[:, -1000:], v[:, -1000:] = kt, vt
    got = W.ops.masked_attn(q, k, v, 0.1, True, doc_starts=_ints([[0, Lk - 1000]]))
    want, tol = _reference(q, kt, vt, 0.1, causal=True)
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.gpu
def test_less_scratch(W):
    """With the scratch of the C call cut short the keys are split less far; without any, not at all."""
    N, lib = W._native, W._native.lib()
    q, k, v, _ = _make(1, 1, 3000, 8, 2, 128, BF, 21)
    need = lib.wan_masked_attn_workspace(1, 8, 2, 1, 3000, 128, None)
    assert need > 0
    want, tol = _reference(q, k, v, 0.1)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    for n in (need, need - 1, need // 2, 9000, 1, 0):
        out = torch.full_like(q, float("nan"))
        N.check("wan_masked_attn", lib.wan_masked_attn(
            N.tensor4(q), N.tensor4(k), N.tensor4(v), N.tensor4(out), 1, 8, 2, 1, 3000, 128, 0, 0.1, None,
            ws.data_ptr() if n else None, n, torch.cuda.current_stream().cuda_stream))
        assert ((out.double() - want).abs() <= tol).all(), n


@pytest.mark.gpu
def test_output_by_strides(W):
    """Rows around the output stay as they were."""
    N, lib = W._native, W._native.lib()
    for Lq in (3, 290):
        q, k, v, _ = _make(2, Lq, 290, 6, 3, 64, HF, 2)
        whole = torch.full((2, Lq + 2, 8, 72), 7.0, device=DEV, dtype=HF)
        out = whole[:, 1:-1, 1:-1, :64]
        N.check("wan_masked_attn", lib.wan_masked_attn(
            N.tensor4(q), N.tensor4(k), N.tensor4(v), N.tensor4(out), 2, 6, 3, Lq, 290, 64, 1, 0.1, None, None, 0,
            torch.cuda.current_stream().cuda_stream))
        want, tol = _reference(q, k, v, 0.1)
        assert ((out.double() - want).abs() <= tol).all()
        out.fill_(7.0)
        assert (whole == 7.0).all()


@pytest.mark.gpu
def test_refusals_and_empty(W):
    q, k, v, bias = _make(2, 5, 9, 4, 2, 64, BF, 1, 3)
    f = W.ops.masked_attn
    i = _ints([1, 2])
    for args, what in (((q.float(), k, v, 0.1), "expected one of"), ((q, k.half(), v, 0.1), "different types"),
                       ((q, k, v[:, :8], 0.1), "differ"), ((q[..., :32], k[..., :32], v[..., :32], 0.1), "head_dim"),
                       ((q[:, :, :3], k, v, 0.1), "disagree"), ((q[:1], k, v, 0.1), "disagree"),
                       ((q, k, v, 0.1, False, 0.0, bias[:, 1:]), "bias"), ((q, k, v, 0.1, False, 0.0, bias[1:]), "bias"),
                       ((q, k, v, 0.1, False, 0.0, bias.half()), "bias"), ((q, k, v, 0.1, False, 0.0, None, i), "doc_starts"),
                       ((q, k, v, 0.1, False, 0.0, None, i.view(2, 1).long()), "doc_starts"),
                       ((q, k, v, 0.1, False, 0.0, None, None, i), "prefix_lens"),
                       ((q, k, v, 0.1, True, 0.0, None, i.view(2, 1), i), "prefix_lens"),
                       ((q, k, v, 0.1, True, 0.0, None, None, None, i[:1]), "seqlen_k"),
                       ((q, k, v, 0.1, True, 0.0, None, None, None, None, i.cpu()), "q_start")):
        with pytest.raises(ValueError, match=what):
            f(*args)
    for args, what in (((q, k, v, -0.1), "softmax_scale"), ((q, k, v, 0.1, False, -2.0), "softcap")):
        with pytest.raises(RuntimeError, match=what):
            f(*args)
    assert f(q[:, :0], k, v, 0.1).shape == (2, 0, 4, 64)
    assert (f(q, k[:, :0], v[:, :0], 0.1) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Lq,Lk", [(1, 1500), (300, 300), (70, 900)])
def test_native_equals_python_and_graph_replays(W, Lq, Lk):
    """The same bits from the native and the Python function, on another stream, and from a captured graph
    replayed on new values with other work in between."""
    f = W.ops.masked_attn

    def make(seed):
        q, k, v, bias = _make(2, Lq, Lk, 4, 2, 64, BF, seed, 50)
        lens = _ints([Lk - 7 * seed, Lk // (seed + 1) + Lq])
        return q, k, v, 0.1, True, 20.0, bias, None, _ints([seed, 3 * seed]), lens, lens - Lq
    args = make(0)
    native = f(*args)
    assert torch.equal(native, f(args[0].detach().requires_grad_(), *args[1:]).detach())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = f(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(native, again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f(*args)
    for seed in (1, 2, 3):
        for t, n in zip(args, make(seed)):
            if isinstance(t, torch.Tensor):
                t.copy_(n)
        want = f(*args)
        torch.randn(100, 100, device=DEV).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_two_streams_at_once(W):
    """Calls that split their keys, side by side on two streams: each has scratch of its own."""
    a, b = (_make(4, 1, 5000, 16, 4, 128, BF, s)[:3] for s in (1, 2))
    want = [W.ops.masked_attn(*x, 0.1) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for n, x in enumerate((a, b)):
            with torch.cuda.stream(streams[n]):
                got[n].append(W.ops.masked_attn(*x, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[n]) for n in range(2) for g in got[n])


@pytest.mark.gpu
@pytest.mark.parametrize("grow", [False, True])
def test_packed_requests_end_to_end(W, grow):
    """Norm and rotation of a packed projection, then the attention within each document, against the same
    documents one by one; and (grow) token by token over a cache against the whole prompt at once."""
    g = torch.Generator(device=DEV).manual_seed(17)
    Hq, Hk, D = 8, 2, 128
    sizes = [70, 1, 130, 99]
    T = sum(sizes)
    x = torch.randn(1, T, (Hq + 2 * Hk) * D, generator=g, device=DEV).to(BF)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in x.split([Hq * D, Hk * D, Hk * D], -1))
    gq, gk = ((1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(BF) for _ in range(2))
    ang = torch.outer(torch.arange(200, device=DEV).float(), 1.0 / 10000 ** (torch.arange(64, device=DEV) / 64))
    rope = (ang.cos(), ang.sin())
    pos = torch.cat([torch.arange(n, device=DEV) for n in sizes]).int()[None]
    qn, kn = W.ops.head_norm_rope(q, k, gq, gk, 1e-6, *rope, pos, False)
    starts = [sum(sizes[:i]) for i in range(len(sizes))]
    out = W.ops.masked_attn(qn, kn, v, D ** -0.5, grow, doc_starts=_ints([starts]))
    want, tol = _reference(qn, kn, v, D ** -0.5, causal=grow, docs=_ints([starts]))
    assert ((out.double() - want).abs() <= tol).all()
    for s, n in zip(starts, sizes):
        at = slice(s, s + n)
        q1, k1 = W.ops.head_norm_rope(q[:, at], k[:, at], gq, gk, 1e-6, *rope, None, False)
        assert torch.equal(q1, qn[:, at]) and torch.equal(k1, kn[:, at])
        if grow:
            cache_k, cache_v = torch.zeros(1, 140, Hk, D, device=DEV, dtype=BF), torch.zeros(1, 140, Hk, D, device=DEV, dtype=BF)
            for i in (0, n // 2, n - 1):
                cache_k[:, :i + 1], cache_v[:, :i + 1] = k1[:, :i + 1], v[:, s:s + i + 1]
                one = W.ops.masked_attn(q1[:, i:i + 1], cache_k, cache_v, D ** -0.5, True, seqlen_k=_ints([i + 1]),
                                        q_start=_ints([i]))
                assert ((one.double() - want[:, s + i:s + i + 1]).abs() <= tol[:, s + i:s + i + 1]).all()
