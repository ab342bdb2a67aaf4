"""Host-side checks of the attention under masks: its launch plan (csrc/plans.h), and as properties of their index
maps the kernel's LDS layouts, the protocol of its rings, its order of workgroups and its blocks of documents
(csrc/masked_attn.h).  No kernel runs here."""
import ctypes
import os
import random
import subprocess

import pytest

import plans

SHIM = """
#include "plans.h"
using namespace wan;
extern "C" void plan(int B, int Hq, int Hk, int Lq, int Lk, int D, int causal, int ragged, int docs, int cus, size_t scratch,
                     long long* out) {
  const MaskedPlan p = masked_plan(B, Hq, Hk, Lq, Lk, D, causal != 0, ragged != 0, docs, cus, scratch);
  const long long v[] = {p.pack, p.block_rows, p.key_groups, p.splits, p.part_rows, p.part_floats, p.blocks, p.out_rows,
                         (long long)p.bytes, p.by_docs};
  for (int i = 0; i < 10; ++i) out[i] = v[i];
}
extern "C" int turn(long long workgroups, int cus) { return masked_turn(workgroups, cus); }
"""
FIELDS = ("pack", "block_rows", "key_groups", "splits", "part_rows", "part_floats", "blocks", "out_rows", "bytes", "by_docs")


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "p.cpp").write_text(SHIM)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", plans.CSRC,
                    str(d / "p.cpp"), "-o", str(d / "p.so")], check=True)
    lib = ctypes.CDLL(str(d / "p.so"))

    def call(B, Hq, Hk, Lq, Lk, D, causal=0, ragged=0, docs=0, scratch=1 << 50, cus=256):
        out = (ctypes.c_longlong * 10)()
        lib.plan(B, Hq, Hk, Lq, Lk, D, causal, ragged, docs, cus, ctypes.c_size_t(scratch), out)
        return dict(zip(FIELDS, out))
    call.lib = lib
    return call


def _sizes(rng, n):
    for _ in range(n):
        Hk = rng.choice([1, 2, 8, 24])
        Lk = rng.choice([0, 1, 63, 64, 65, 1000, 4096, 100000])
        yield (rng.choice([1, 2, 16, 64]), Hk * rng.choice([1, 3, 4, 8, 29, 32, 40, 64]), Hk,
               rng.choice([1, 2, 7, 33, 256, 257, max(1, Lk)]), Lk, rng.choice([64, 128]), rng.randint(0, 1), rng.randint(0, 1),
               rng.choice([0, 0, 1, 5, 64, 300]))


def test_plan_covers_the_rows_within_its_scratch(plan, W):
    rng = random.Random(1)
    ws = W._native.lib().wan_masked_attn_workspace
    for s in _sizes(rng, 3000):
        B, Hq, Hk, Lq, Lk, D, causal, ragged, docs = s
        free = plan(*s)
        mask = W._native.WanAttnMask(causal=causal, seqlen_k=256 * ragged, doc_starts=256 * (docs > 0), docs=docs)
        assert free["bytes"] == ws(B, Hq, Hk, Lq, Lk, D, ctypes.byref(mask)), s        # (256 CUs without a device)
        for scratch in (0, free["bytes"] // 3, max(free["bytes"] - 1, 0), free["bytes"]):
            p = plan(*s, scratch=scratch)
            units = B * (Hq // p["pack"])
            assert p["bytes"] <= scratch and (p["splits"] > 1) == (p["bytes"] > 0)
            assert (Hq // Hk) % p["pack"] == 0 and p["pack"] <= 28 and p["out_rows"] == B * Lq * Hq
            assert p["block_rows"] in ((32,) if Lq * p["pack"] <= 32 else (128, 256)) and 1 <= p["splits"] <= 64
            plain = -(-Lq * p["pack"] // p["block_rows"])
            assert p["blocks"] >= plain * units and (p["by_docs"] or p["blocks"] == plain * units)
            assert p["by_docs"] == (docs > 0 and p["splits"] == 1 and p["block_rows"] > 32)
            if p["splits"] > 1:
                assert p["part_rows"] == min(Lq * p["pack"], p["block_rows"]) and p["part_floats"] % 4 == 0
                assert p["part_floats"] >= p["part_rows"] * (D + 2)
                assert p["bytes"] == p["blocks"] * p["splits"] * p["part_floats"] * 4


def test_division_by_a_product():
    """FastDiv: n / d as (n * m) >> (31 + s)."""
    rng = random.Random(2)
    for d in list(range(1, 2000)) + [rng.randint(1, 2 ** 31 - 1) for _ in range(5000)] + [2 ** k + e for k in range(1, 31) for e in (-1, 0, 1)]:
        s = max(0, (d - 1).bit_length())
        m = -(-(1 << (31 + s)) // d)
        assert m < 2 ** 32
        top = (2 ** 31 - 1) // d * d
        for n in (0, 1, d - 1, d, d + 1, top - 1, top, 2 ** 31 - 1, rng.randint(0, 2 ** 31 - 1)):
            if 0 <= n < 2 ** 31:
                assert (n * m) >> (31 + s) == n // d, (n, d)


# ─── the blocks of documents ──────────────────────────────────────────────────

def _runs(starts, start, Lq, pack, BM, chunk=64):
    """RowBlock's runs of a unit, (first row, end), in the order that the kernel gives them blocks."""
    rows, out, begun = Lq * pack, [], 0
    for j0 in range(0, len(starts) + 1, chunk):
        to = []
        for j in range(j0, j0 + chunk):
            to.append(min(max(starts[j] - start, 0), Lq) * pack if j < len(starts) else rows)
        for i in range(1, chunk):
            to[i] = max(to[i], to[i - 1])
        to = [max(begun, t) for t in to]
        frm = [begun] + to[:-1]
        large = [t - f >= 2 * BM for f, t in zip(frm, to)]
        heads = [i for i in range(chunk) if i == 0 or large[i] or large[i - 1]]
        part = []
        for n, i in enumerate(heads):
            # (the kernel takes the end from the next head's own lane: its documents before it have ended there)
            later = heads[n + 1] if n + 1 < len(heads) else None
            part.append((frm[i], frm[later] if later is not None else to[-1]))
        out += sorted(part, key=lambda r: (-(r[1] - r[0]), r[0]))
        begun = to[-1]
    return out


@pytest.mark.parametrize("BM", [128, 256])
def test_blocks_of_documents_hold_every_row_once(plan, BM):
    rng = random.Random(BM)
    for trial in range(400):
        Lq, pack = rng.choice([1, 5, 300, 3000, 8192]), rng.choice([1, 2, 8])
        n = rng.choice([1, 2, 6, 63, 64, 65, 200])
        starts = [rng.randint(-10, Lq + 10) for _ in range(n)]
        if trial % 4:
            starts.sort()
        start = rng.choice([0, 0, 50, -20])
        runs = _runs(starts, start, Lq, pack, BM)
        pos = sorted(r for r in runs if r[1] > r[0])
        assert [r[0] for r in pos] == [0] + [r[1] for r in pos[:-1]] and pos[-1][1] == Lq * pack
        blocks = sum(-(-(e - f) // BM) for f, e in runs)
        plain = -(-Lq * pack // BM)
        assert blocks <= plain + min(plain + 2 + n // 64, n + 1), (starts, Lq, pack)     # what the plan launches


# ─── LDS ──────────────────────────────────────────────────────────────────────

def k_swz(HD, row):
    return row & 15 if HD == 128 else (row >> 1) & 7


def v_swz(HD, row):
    return (row & 3) << 2 if HD == 128 else (row & 2) << 1


@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("keys,waves", [(32, 1), (64, 8), (64, 4)])
def test_tile_copies_and_reads(HD, keys, waves):
    cpr, rows_kb = HD // 8, 512 // HD
    per = keys // rows_kb // waves
    assert per * rows_kb * waves == keys
    for swz in (k_swz, v_swz):
        lds = {}
        for wave in range(waves):
            for u in range(per):
                for lane in range(64):
                    row = rows_kb * (wave + waves * u) + lane // cpr
                    at = (wave + waves * u) * 1024 + lane * 16
                    assert at not in lds
                    lds[at] = (row, (lane % cpr) ^ swz(HD, row))
        assert sorted(lds) == list(range(0, keys * HD * 2, 16))
        for row in range(keys):
            for c in range(cpr):
                assert lds[row * HD * 2 + ((c ^ swz(HD, row)) << 4)] == (row, c)
    # k: a phase reads one chunk of 16 rows, on 16 distinct bank groups
    for c in range(cpr):
        for r0 in range(0, keys, 16):
            assert len({(r * HD * 2 + ((c ^ k_swz(HD, r)) << 4)) % 256 for r in range(r0, r0 + 16)}) == 16
    # v: a transposed read takes 4 chunks of 4 rows, and its lanes name each channel's keys in the accumulator's order
    for md in range(HD // 32):
        for r0 in range(0, keys, 4):
            assert len({(r * HD * 2 + (((4 * md + c) ^ v_swz(HD, r)) << 4)) % 256 for r in range(r0, r0 + 4) for c in range(4)}) == 16


@pytest.mark.parametrize("KG", [1, 2])
def test_ring_protocol(KG):
    """Every read finds its tile landed and published by a barrier, and no copy goes into a slot that a slower wave may
    still read: between two barriers all waves' reads may come before or after all copies."""
    def run(nt, mistake=0):
        landed, pending = {"k": {}, "v": {}}, []
        reads = {"k": set(), "v": set()}          # slots read since the last barrier
        writes = {"k": set(), "v": set()}

        def copy(kind, u, clamp):
            if u >= nt and not clamp:
                return
            slot = u % 4
            assert slot not in reads[kind], "overwritten while it may be read"
            writes[kind].add(slot)
            pending.append((kind, slot, min(u, nt - 1) if clamp else u))

        def barrier():
            for kind, slot, u in pending:
                landed[kind][slot] = u
            pending.clear()
            for d in (reads, writes):
                d["k"].clear()
                d["v"].clear()

        def read(kind, u):
            assert landed[kind].get(u % 4) == u, "not there"
            assert u % 4 not in writes[kind], "read while it may be overwritten"
            reads[kind].add(u % 4)
        for u in range(2 + KG):
            copy("k", u, False)
            if u < 2:
                copy("v", u, False)
        barrier()
        for g in range(KG):
            if g < nt:
                read("k", g)
        barrier()
        for u0 in range(0, nt, KG):
            lean = u0 % (2 * KG) == 0 and u0 + 2 * KG + KG <= nt or u0 % (2 * KG) != 0 and u0 + 2 * KG <= nt
            for u in range(u0, u0 + KG):
                if u + KG < nt:
                    read("k", u + KG)
                if u < nt:
                    read("v", u)
            if KG == 2 or u0 % 2 == 0:
                copy("k", u0 + 2 + KG - mistake, lean)
                copy("k", u0 + 3 + KG, lean)
                copy("v", u0 + 2, lean)
                copy("v", u0 + 3, lean)
            if KG == 2 or u0 % 2:
                barrier()
    for nt in range(1, 40):
        run(nt)
    with pytest.raises(AssertionError):
        run(20, mistake=1)


def test_order_reaches_every_block_once():
    for ups, blocks in ((1, 1), (8, 65), (24, 31), (31, 7), (32, 4), (33, 5), (128, 2), (70, 3)):
        seen = set()
        for i in range(ups * blocks):
            group = i // 32 // blocks
            inside = i - group * 32 * blocks
            whole = (group + 1) * 32 <= ups
            size = 32 if whole else ups - group * 32
            at = inside // size
            seen.add((group * 32 + inside - at * size, at))
        assert seen == {(u, a) for u in range(ups) for a in range(blocks)}


@pytest.mark.parametrize("cus", [256, 304, 8, 100])
def test_turned_workgroups_stay_an_order(plan, cus):
    turn = plan.lib.turn
    turn.argtypes = [ctypes.c_longlong, ctypes.c_int]
    for n in (1, cus - 1, cus, cus + 1, cus + 8, 2 * cus - 1, 2 * cus, 2 * cus + 5, 3 * cus - 1, 3 * cus, 1 << 22):
        eights = turn(n, cus)
        assert 0 <= eights <= cus // 8 and cus + 8 * eights <= max(n, cus)
        ids = []
        for i in range(min(n, 4 * cus)):
            turned = (i - cus) >> 3
            ids.append(cus + (eights - 1 - turned) * 8 + (i & 7) if 0 <= turned < eights else i)
        assert sorted(ids) == list(range(len(ids)))
        assert all(a % 8 == b % 8 for a, b in zip(ids, range(len(ids))))      # on the XCD of before
