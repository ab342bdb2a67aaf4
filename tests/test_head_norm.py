"""ops.head_norm_rope: RMSNorm of every q and k head with the rotation, against the formula in 64 bits;
its refusals and its launch plan on the CPU."""
import ctypes
import os
import subprocess

import pytest
import torch

import plans

DEV = "cuda"
STEP = {torch.bfloat16: 2 ** -8, torch.float16: 2 ** -11, torch.float32: 2 ** -24}
# half the distance of the smallest values of each type
SMALL = {torch.bfloat16: 2 ** -134, torch.float16: 2 ** -25, torch.float32: 2 ** -150}


# ─── on the CPU ───────────────────────────────────────────────────────────────

SHIM = """
#include "plans.h"
using namespace wan;
extern "C" {
int chunks(long long tokens, int heads, int lanes) { return head_norm_chunks(tokens, heads, lanes); }
void plan(long long tokens, int heads, int lanes, int n, int* out, long long* waves) {
  const HeadNormPlan p = head_norm_plan(tokens, heads, lanes, n);
  out[0] = p.waves_per_token; out[1] = p.slot_shift; out[2] = p.token_shift;
  *waves = p.waves;
}
}
"""


@pytest.fixture(scope="module")
def plan_lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "p.cpp").write_text(SHIM)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", plans.CSRC,
                    str(d / "p.cpp"), "-o", str(d / "p.so")], check=True)
    return ctypes.CDLL(str(d / "p.so"))


@pytest.mark.parametrize("lanes", [8, 16, 32])
@pytest.mark.parametrize("heads", [1, 2, 3, 5, 8, 20, 40, 48, 65])
def test_plan_reaches_every_head_once(plan_lib, lanes, heads):
    """The kernel's index arithmetic over the launcher's plan: each (token, head) belongs to one lane group."""
    for tokens in (1, 2, 7, 33, 5000):
        n = plan_lib.chunks(ctypes.c_longlong(tokens), heads, lanes)
        assert 1 <= n <= 4
        out, waves = (ctypes.c_int * 3)(), ctypes.c_longlong()
        plan_lib.plan(ctypes.c_longlong(tokens), heads, lanes, n, out, ctypes.byref(waves))
        wpt, slot_shift, token_shift = out
        assert (1 << (slot_shift + token_shift)) * lanes == 64
        per_step, seen = 1 << slot_shift, set()
        groups = waves.value // wpt
        for wave in list(range(min(waves.value, 64))) + list(range(max(0, waves.value - 64), waves.value)):
            group, part = divmod(wave, wpt)
            for slot in range(64 // lanes):
                tok = (group << token_shift) + (slot >> slot_shift)
                for i in range(n):
                    h = part * per_step * n + (slot & (per_step - 1)) + i * per_step
                    if tok < tokens and h < heads:
                        assert (tok, h, wave) in seen or not any((tok, h, w) in seen for w in (wave - 1, wave + 1))
                        seen.add((tok, h, wave))
        assert groups << token_shift >= tokens > (groups - 1) << token_shift
        if waves.value <= 64:
            assert {(t, h) for t, h, _ in seen} == {(t, h) for t in range(tokens) for h in range(heads)}
            assert len(seen) == tokens * heads


def test_abi_refusals(W):
    N = W._native
    lib, t = N.lib(), N.WanTensor(64, 4096, 512, 64)
    P = 256         # an aligned stand-in address: every call fails before a launch

    def call(q=t, k=t, q_out=P, k_out=P, B=1, L=8, Hq=4, Hk=2, D=64, dtype=0, gq=P, gk=P, eps=1e-6, cos=P, sin=P,
             rows=8, pairs=32, pos=None, inter=1):
        rc = lib.wan_head_norm_rope(q, k, q_out, k_out, B, L, Hq, Hk, D, dtype, gq, gk, eps, cos, sin, rows, pairs, pos,
                                    inter, None)
        return rc, N.last_error() if rc else ""

    for kw, code, what in ((dict(B=-1), 1, "negative"), (dict(D=60), 2, "head_dim"), (dict(D=264), 2, "head_dim"),
                           (dict(D=0), 2, "head_dim"), (dict(dtype=3), 2, "dtype"), (dict(B=65536, L=65536), 2, "too many"),
                           (dict(q=N.WanTensor(66, 4096, 512, 64)), 1, "aligned"),
                           (dict(k=N.WanTensor(64, 4096, 516, 64)), 1, "stride"), (dict(q=N.WanTensor(0, 0, 0, 0)), 1, "NULL"),
                           (dict(q_out=None), 1, "q_out"), (dict(k_out=P + 2), 1, "aligned"), (dict(gq=None), 1, "gamma"),
                           (dict(gk=P + 8), 1, "gamma"), (dict(eps=-1.0), 1, "eps"), (dict(eps=float("nan")), 1, "eps"),
                           (dict(sin=None), 1, "both"), (dict(cos=None, sin=None, pos=P), 1, "without tables"),
                           (dict(cos=P + 4), 1, "aligned"), (dict(pairs=0), 2, "rope_pairs"), (dict(pairs=6), 2, "rope_pairs"),
                           (dict(pairs=36), 2, "rope_pairs"), (dict(pairs=12, inter=0), 2, "rope_pairs"),
                           (dict(rows=7), 1, "rows"), (dict(rows=0, pos=P), 1, "rows")):
        rc, msg = call(**kw)
        assert rc == code and what in msg and msg.startswith("wan_head_norm_rope"), (kw, rc, msg)
    assert call(B=0)[0] == call(L=0)[0] == call(Hq=0, Hk=0)[0] == 0


def test_operator_refuses_host_tensors_and_traces(W):
    x = torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        W.ops.head_norm_rope(x, x, x[0, 0, 0], x[0, 0, 0], 1e-6)
    q, k = torch.empty(2, 5, 6, 96, device="meta"), torch.empty(2, 5, 3, 96, device="meta")
    a, b = torch.ops.wan_hip.head_norm_rope(q, k, q, q, 1e-6)
    assert a.shape == q.shape and b.shape == k.shape


# ─── on the GPU ───────────────────────────────────────────────────────────────

def _make(B, L, Hq, Hk, D, dtype, seed, P=0, rows=None, positions=False):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=g, device=DEV)
    x = (normal(B, L, (Hq + Hk) * D) * (0.2 + normal((Hq + Hk) * D).abs())).to(dtype)
    q, k = (t.unflatten(-1, (-1, D)) for t in x.split([Hq * D, Hk * D], -1))        # views of one projection
    gq, gk = ((1 + normal(D)).to(dtype) for _ in range(2))
    if not P:
        return q, k, gq, gk, 1e-6
    rows = L if rows is None else rows
    ang = torch.rand(rows, P, generator=g, device=DEV) * 6.3
    pos = torch.randint(0, rows, (B, L), generator=g, device=DEV, dtype=torch.int32) if positions else None
    return q, k, gq, gk, 1e-6, ang.cos(), ang.sin(), pos


def _want(x, gamma, eps, cos=None, sin=None, pos=None, interleaved=True):
    """(the formula in 64 bits, the length of each value's pair)"""
    y = x.double() / (x.double().square().mean(-1, keepdim=True) + eps).sqrt() * gamma.double()
    if cos is None:
        return y, y.abs()
    P = cos.shape[1]
    at = torch.arange(x.shape[1], device=x.device).expand(x.shape[:2]) if pos is None else pos.long()
    c, s = (t.double()[at][:, :, None] for t in (cos, sin))
    i, j = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    out, size = y.clone(), y.abs()
    out[..., i], out[..., j] = y[..., i] * c - y[..., j] * s, y[..., i] * s + y[..., j] * c
    size[..., i] = size[..., j] = (y[..., i].square() + y[..., j].square()).sqrt()
    return out, size


def _close(got, want, size, D):
    """One rounding of the result, and before it in fp32: D products and sums of the squares (half of their
    relative error in the root), the division, root and two products (4), the rotation's two products and
    sum (3 more of the pair's length, whose cos + sin is at most 1.42), each 2^-24 at most."""
    t = STEP[got.dtype]
    before = size * (D / 2 + 10) * 2 ** -24
    assert ((got.double() - want).abs() <= (want.abs() + before) * t + before + SMALL[got.dtype]).all()


def _check(args, interleaved=True):
    W_ops, q, k, gq, gk, eps, *rope = args
    full = (*rope, *[None] * (3 - len(rope)))
    got = W_ops.head_norm_rope(q, k, gq, gk, eps, *full, interleaved)
    for out, x, gamma in zip(got, (q, k), (gq, gk)):
        assert out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous()
        _close(out, *_want(x, gamma, eps, *full, interleaved), x.shape[-1])
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("B,L,Hq,Hk,D", [(1, 1, 1, 1, 64), (8, 1, 32, 8, 128), (2, 37, 24, 24, 128), (3, 5, 3, 1, 8),
                                         (1, 700, 5, 2, 96), (2, 33, 7, 7, 256), (1, 129, 2, 1, 200), (1, 3000, 16, 4, 64),
                                         (1, 4099, 6, 6, 256)])
def test_norm_alone(W, B, L, Hq, Hk, D, dtype):
    _check((W.ops, *_make(B, L, Hq, Hk, D, dtype, B * L + D)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(STEP))
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("B,L,Hq,Hk,D,P", [(8, 1, 32, 8, 128, 64), (2, 37, 24, 24, 128, 64), (3, 517, 16, 4, 64, 16),
                                           (1, 70, 3, 2, 96, 48), (1, 70, 3, 2, 96, 24), (2, 9, 4, 1, 256, 128),
                                           (1, 1, 1, 1, 64, 8), (1, 2160, 24, 24, 128, 64)])
@pytest.mark.parametrize("positions", [True, False])
def test_norm_and_rotation(W, B, L, Hq, Hk, D, P, interleaved, positions, dtype):
    _check((W.ops, *_make(B, L, Hq, Hk, D, dtype, L + P, P, L + 13, positions)), interleaved)


@pytest.mark.gpu
def test_positions_outside_the_tables_give_nan_and_nothing_else(W):
    q, k, gq, gk, eps, cos, sin, pos = _make(2, 40, 5, 2, 128, torch.bfloat16, 3, 32, 50, True)
    good = W.ops.head_norm_rope(q, k, gq, gk, eps, cos, sin, pos)
    bad = pos.clone()
    for (b, l), p in (((0, 0), -1), ((0, 39), 50), ((1, 7), 2 ** 31 - 1), ((1, 8), -2 ** 31)):
        bad[b, l] = p
    for a, w in zip(W.ops.head_norm_rope(q, k, gq, gk, eps, cos, sin, bad), good):
        hit = (bad != pos)[:, :, None, None].expand_as(a)
        assert a[hit].isnan().all() and torch.equal(a[~hit], w[~hit])


@pytest.mark.gpu
def test_values_stay_in_their_head(W):
    """NaN, infinities and zeros of one head reach no other head or token."""
    q, k, gq, gk, eps, cos, sin, _ = _make(1, 6, 4, 4, 64, torch.bfloat16, 5, 32)
    good = W.ops.head_norm_rope(q, k, gq, gk, eps, cos, sin)
    q, k = q.clone(), k.clone()
    q[0, 2, 1, 5], q[0, 3, 0, 0], k[0, 4, 3] = float("nan"), float("inf"), 0
    got = W.ops.head_norm_rope(q, k, gq, gk, eps, cos, sin)
    assert got[0][0, 2, 1].isnan().all() and got[0][0, 3, 0].isnan().any() and (got[1][0, 4, 3] == 0).all()
    same = torch.ones(6, 4, dtype=torch.bool)
    same[2, 1] = same[3, 0] = False
    assert torch.equal(got[0][0][same], good[0][0][same])


@pytest.mark.gpu
def test_strides(W):
    """[B, heads, L, D] caches, broadcast batches and padded rows."""
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(2, 6, 50, 136, generator=g, device=DEV).half()
    q, k = x[:, :4, :, :128].transpose(1, 2), x[:1, 4:, 3:, 8:].transpose(1, 2).expand(2, -1, -1, -1)
    gq = torch.rand(128, generator=g, device=DEV).half()
    got = W.ops.head_norm_rope(q[:, 3:], k, gq, gq, 1e-5)
    _close(got[0], *_want(q[:, 3:], gq, 1e-5), 128)
    _close(got[1], *_want(k, gq, 1e-5), 128)


@pytest.mark.gpu
def test_refusals_and_empty(W):
    q, k, gq, gk, eps, cos, sin, pos = _make(2, 6, 4, 2, 64, torch.bfloat16, 5, 32, 9, True)
    f = W.ops.head_norm_rope
    for args, what in (((q.double(), k, gq, gk, eps), "expected one of"), ((q, k.float(), gq, gk, eps), "disagree"),
                       ((q, k[:, :3], gq, gk, eps), "disagree"), ((q[..., :60], k[..., :60], gq, gk, eps), "head_dim"),
                       ((q, k, gq[1:], gk, eps), "gamma_q"), ((q, k, gq, gk.float(), eps), "gamma_k"),
                       ((q, k, gq, gk, eps, cos), "both"), ((q, k, gq, gk, eps, None, None, pos), "positions"),
                       ((q, k, gq, gk, eps, cos, sin.half(), pos), "sin"), ((q, k, gq, gk, eps, cos, sin[:5], pos), "alike"),
                       ((q, k, gq, gk, eps, cos, sin, pos.long()), "positions"),
                       ((q, k, gq, gk, eps, cos, sin, pos[:, :5]), "positions"),
                       ((q[0], k[0], gq, gk, eps), "expected"), ((q[..., ::2], k[..., ::2], gq[:32], gk[:32], eps), "contiguous")):
        with pytest.raises(ValueError, match=what):
            f(*args)
    for args, what in (((q, k, gq, gk, eps, cos[:5].contiguous(), sin[:5].contiguous()), "5 rows for 6 tokens"),
                       ((q, k, gq, gk, eps, cos[:, :30].contiguous(), sin[:, :30].contiguous(), pos), "rope_pairs"),
                       ((q, k, gq, gk, -1.0), "eps")):
        with pytest.raises(RuntimeError, match=what):
            f(*args)
    a, b = f(q[:, :0], k[:, :0], gq, gk, eps)
    assert a.shape == (2, 0, 4, 64) and b.shape == (2, 0, 2, 64)


@pytest.mark.gpu
def test_native_equals_python_and_graph_replays(W):
    args = _make(2, 65, 6, 2, 128, torch.bfloat16, 9, 64, 80, True)
    native = W.ops.head_norm_rope(*args, False)
    python = W.ops.head_norm_rope(args[0].detach().requires_grad_(), *args[1:], False)
    assert all(torch.equal(a, b.detach()) for a, b in zip(native, python))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        W.ops.head_norm_rope(*args, False)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = W.ops.head_norm_rope(*args, False)
    for seed in (1, 2, 3):
        for t, n in zip(args, _make(2, 65, 6, 2, 128, torch.bfloat16, seed, 64, 80, True)):
            if isinstance(t, torch.Tensor):
                t.copy_(n)
        want = W.ops.head_norm_rope(*args, False)
        torch.randn(100, 100, device=DEV).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
