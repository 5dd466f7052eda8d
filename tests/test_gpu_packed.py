"""Attention over packed prompts (pkv.attn_packed) against the formula in 64
bits, on the GPU.

Bound per element, from the kernel's arithmetic with u half a step of the row
type (2^-8 bf16, 2^-11 fp16) and A = sum_j w_j |v_j| of the softmax weights w:
  u A         the weights rounded for the second product
  u |out|     their sum (of the same rounded weights), u |out| the output's own rounding; below the type's smallest
              normal number (2^-14 in fp16) the spacing stays that number's: u times it (2^-25)
  e (A + |out|)   scores in f32: a dot product of D terms is off by at most (D + 16) 2^-24 scale sum |q k|
              (S, its largest over the row's keys), twice that in a ratio of weights, and 2^-20 for exp2, the
              sigmoid and the division
  n 2^-24 A   n weighted values added up in f32
  fp16: weights below 2^-14 are multiples of 2^-24, off by 2^-25 at most: n 2^-25 max |v| (the largest weight is 1
        or more).
"""
import numpy as np
import pytest
import torch

import pkv

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def offsets(lens, lead=0):
    return np.concatenate([[lead], lead + np.cumsum(lens)]).astype(np.int32)


def inputs(lens, Hq, Hkv, D, dtype, seed, dev, gate=False, lead=0, tail=0, amp=1.5):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    T = int(sum(lens)) + lead + tail
    r = lambda H, a: (torch.randn(T, H, D, device=dev, generator=g) * a).to(TYPES[dtype])
    return dict(q=r(Hq, amp), k=r(Hkv, amp), v=r(Hkv, 1.0), gate=r(Hq, 2.0) if gate else None,
                cu=torch.from_numpy(offsets(lens, lead)).to(dev), lens=list(lens), lead=lead, scale=D ** -0.5)


def reference(c):
    """out and its bound in float64, rows outside the sequences NaN."""
    q, k, v = (c[n].double() for n in ("q", "k", "v"))
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    u = torch.finfo(c["q"].dtype).eps / 2
    out = torch.full((T, Hq, D), float("nan"), dtype=torch.float64, device=q.device)
    tol = out.clone()
    a = c["lead"]
    for n in c["lens"]:
        for h in range(Hq if n else 0):
            qq, kk, vv = q[a:a + n, h], k[a:a + n, h // G], v[a:a + n, h // G]
            seen = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
            x = torch.where(seen, qq @ kk.t().contiguous() * c["scale"], -float("inf"))
            w = torch.softmax(x, -1)
            o, A = w @ vv, w @ vv.abs()
            S = torch.where(seen, qq.abs() @ kk.abs().t().contiguous() * c["scale"], 0).amax(-1, keepdim=True)
            e = 2 * (D + 16) * 2.0 ** -24 * S + 2.0 ** -20
            m = torch.arange(1, n + 1, device=q.device, dtype=torch.float64)[:, None]
            low = m * 2.0 ** -25 * vv.abs().amax() if c["q"].dtype is torch.float16 else 0
            t = (u + e + m * 2.0 ** -24) * A + (u + e) * o.abs() + low
            sig = torch.sigmoid(c["gate"][a:a + n, h].double()) if c["gate"] is not None else 1.0
            out[a:a + n, h] = o * sig
            tol[a:a + n, h] = t * sig + u * (o * sig).abs() + torch.finfo(c["q"].dtype).tiny * u
        a += n
    return out, tol


def run(c, out=None, **kw):
    if out is None:
        out = torch.full_like(c["q"], 7.0)
    pkv.attn_packed(c["q"], c["k"], c["v"], c["cu"], out, c["scale"], gate=c["gate"], **kw)
    return out


def check(c, got, what=""):
    want, tol = reference(c)
    rows = slice(c["lead"], c["lead"] + sum(c["lens"]))
    err = (got[rows].double() - want[rows]).abs()
    worst = float((err / tol[rows]).max()) if err.numel() else 0.0
    print(f"{what}: {err.numel()} elements, worst error over bound {worst:.3f}", flush=True)
    assert worst <= 1.0 and not torch.isnan(got[rows]).any()


def check_fast(c):
    """check() for many sequences: those of a length at once."""
    got, at = run(c), np.cumsum([c["lead"]] + c["lens"])
    D, G = c["q"].shape[2], c["q"].shape[1] // c["k"].shape[1]
    u, worst = torch.finfo(c["q"].dtype).eps / 2, 0.0
    for n in sorted(set(c["lens"]) - {0}):
        starts = torch.from_numpy(np.flatnonzero(np.array(c["lens"]) == n)).to(got.device)
        rows = torch.from_numpy(at).to(got.device)[starts][:, None] + torch.arange(n, device=got.device)
        for part in rows.split(max(1, 20000 // (n * n) + 1)):
            # [sequences, heads, rows, dims]
            q, o = (x[part].double().transpose(1, 2) for x in (c["q"], got))
            k, v = (x[part].double().transpose(1, 2).repeat_interleave(G, 1) for x in (c["k"], c["v"]))
            kt, seen = k.transpose(2, 3).contiguous(), torch.ones(n, n, dtype=torch.bool, device=got.device).tril()
            w = torch.softmax(torch.where(seen, q @ kt * c["scale"], -float("inf")), -1)
            S = torch.where(seen, q.abs() @ kt.abs() * c["scale"], 0).amax(-1, keepdim=True)
            e = 2 * (D + 16) * 2.0 ** -24 * S + 2.0 ** -20
            want, A = w @ v, w @ v.abs()
            m = torch.arange(1, n + 1, device=got.device, dtype=torch.float64)[:, None]
            tol = (u + e + m * 2.0 ** -24) * A + (2 * u + e) * want.abs()
            err = ((o - want).abs() / tol).max()
            assert not torch.isnan(o).any()
            worst = max(worst, float(err))
    print(f"{len(c['lens'])} sequences: worst error over bound {worst:.3f}", flush=True)
    assert worst <= 1.0
    end = c["lead"] + sum(c["lens"])
    assert (got[:c["lead"]] == 7).all() and (got[end:] == 7).all()


LENS = [[1], [2, 1, 0, 5], [31, 32, 33, 0], [63, 64, 65, 127, 128, 129], [300, 1, 700], [1025]]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (6, 6), (14, 2), (20, 4)])
def test_rows_match_the_formula(dev, dtype, D, Hq, Hkv):
    for i, lens in enumerate(LENS):
        print("case", dtype, D, Hq, Hkv, lens, flush=True)
        c = inputs(lens, Hq, Hkv, D, dtype, 100 * i + D + Hq, dev, gate=i % 2 == 1)
        check(c, run(c), f"{dtype} D {D} heads {Hq}/{Hkv} lens {lens}")


@pytest.mark.parametrize("G", [1, 2, 3, 5, 8, 16, 40])
def test_any_group(dev, G):
    print("case group", G, flush=True)
    c = inputs([77, 130, 3], 2 * G, 2, 64, "bf16", G, dev)
    check(c, run(c), f"G {G}")


@pytest.mark.parametrize("D", [64, 128, 256])
def test_long_prompts_and_many_sequences(dev, D):
    for lens, Hq, Hkv in (([5000], 2, 1), ([1 + 7 * i % 50 for i in range(700)], 4, 2),
                          ([1 + 37 * i % 211 for i in range(256)], 5, 1), ([1 + 37 * i % 211 for i in range(257)], 5, 1),
                          ([500, 3, 0, 900, 0, 0, 1300, 65], 8, 2)):
        print("case", D, len(lens), flush=True)
        c = inputs(lens, Hq, Hkv, D, "bf16", D, dev)
        check(c, run(c), f"D {D}, {len(lens)} sequences")


def test_views_of_a_projection_row(dev):
    """q and gate inside [Hq x (q | gate) | k | v] rows, out head-major and inside wider rows."""
    lens, Hq, Hkv, D = [40, 100, 7], 8, 2, 128
    T = sum(lens)
    x = (torch.randn(T, (2 * Hq + 2 * Hkv) * D, device=dev, generator=torch.Generator(dev).manual_seed(3))).bfloat16()
    qg = x[:, :2 * Hq * D].view(T, Hq, 2, D)
    c = dict(q=qg[:, :, 0], gate=qg[:, :, 1], k=x[:, 2 * Hq * D:(2 * Hq + Hkv) * D].view(T, Hkv, D),
             v=x[:, (2 * Hq + Hkv) * D:].view(T, Hkv, D), cu=torch.from_numpy(offsets(lens)).to(dev), lens=lens, lead=0,
             scale=D ** -0.5)
    major = torch.full((Hq, T, D), 7.0, device=dev, dtype=torch.bfloat16)
    run(c, major.transpose(0, 1))
    check(c, major.transpose(0, 1), "head-major out")
    wide = torch.full((T, Hq, 3, D), 7.0, device=dev, dtype=torch.bfloat16)
    run(c, wide[:, :, 1])
    assert torch.equal(wide[:, :, 1], major.transpose(0, 1)) and (wide[:, :, 0::2] == 7).all()
    # one kv head for all, by a stride of 0
    c["k"], c["v"] = c["k"][:, :1].expand(T, 2, D), c["v"][:, :1].expand(T, 2, D)
    check(c, run(c), "broadcast kv heads")


@pytest.mark.parametrize("more", [[], [129] * 60, [1] * 300 + [129] * 60])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_outside_the_sequences(dev, D, more):
    """Rows before the first and behind the last sequence, NaN in them: neither read into others nor written."""
    c = inputs([70, 0, 33] + more, 4, 2, D, "bf16", 5, dev, gate=True, lead=9, tail=50)
    n = 103 + sum(more)
    inner = slice(9, 9 + n)
    clean = run(c)
    for x in ("q", "k", "v", "gate"):
        keep = c[x][inner].clone()
        c[x].fill_(float("nan"))
        c[x][inner] = keep
    got = run(c)
    assert torch.equal(got[inner], clean[inner])
    assert (got[:9] == 7).all() and (got[9 + n:] == 7).all()


@pytest.mark.parametrize("more", [[], [129] * 40, [1] * 300 + [129] * 40])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_infinite_and_nan_values_reach_the_rows_that_attend_them(dev, D, dtype, more):
    """Alone (few tiles), and in batches of many tiles and many sequences."""
    lens, Hq, Hkv = [150, 40] + more, 6, 2
    c = inputs(lens, Hq, Hkv, D, dtype, 11, dev)
    clean = run(c)
    inf = float("inf")
    for at, x in ((3, inf), (37, -inf), (38, float("nan")), (100, inf), (101, -inf), (149, float("nan"))):
        y = dict(c, v=c["v"].clone())
        y["v"][at, 1, 5] = x
        got = run(y)
        # what does not attend it: earlier rows, the other sequence, other kv heads and dims
        same = torch.ones_like(got, dtype=torch.bool)
        same[at:150, 3:, 5] = False
        assert torch.equal(got[same], clean[same]), (at, x)
        hit = got[at:150, 3:, 5]
        # (an fp16 weight below 2^-25 is 0, and 0 x infinity NaN)
        assert (torch.isnan(hit) if x != x else (hit == x) | (torch.isnan(hit) & (dtype == "fp16"))).all(), (at, x)
    # both signs: NaN from the row on that attends both
    y = dict(c, v=c["v"].clone())
    y["v"][100, 0, 0], y["v"][101, 0, 0] = inf, -inf
    got = run(y)
    assert not torch.isfinite(got[100, :3, 0]).any() and torch.isnan(got[101:150, :3, 0]).all()
    assert torch.equal(got[:100], clean[:100])
    # keys: a NaN key makes the rows that attend it NaN, an infinite one decides or drops out
    y = dict(c, k=c["k"].clone())
    y["k"][60, 0] = float("nan")
    got = run(y)
    assert torch.equal(got[:60], clean[:60]) and torch.isnan(got[60:150, :3]).all()
    assert torch.equal(got[:, 3:], clean[:, 3:]) and torch.equal(got[150:], clean[150:])
    # a query: its own row
    y = dict(c, q=c["q"].clone())
    y["q"][20, 2, 0] = inf
    got = run(y)
    same = torch.ones(got.shape[:2], dtype=torch.bool, device=dev)
    same[20, 2] = False
    assert torch.equal(got[same], clean[same])


def test_gates_at_their_ends(dev):
    """Gates that close a row, open it, are infinite or NaN, and one on an infinite value. Below -87.3 the result is 0,
    within 1.2e-38 of the value: the bound's smallest term is below that, so those two dims are held to it alone."""
    c = inputs([60], 4, 2, 64, "bf16", 12, dev, gate=True)
    ends = torch.tensor([-87.0, -86.5, -80.0, -60.0, -30.0, 0.0, 20.0, 88.0, 3e38], device=dev).bfloat16()
    c["gate"][:, :, :9] = ends
    plain = run(dict(c, gate=None))
    got = run(c)
    check(c, got, "gates")
    # (0.01 e^-87 is above 2^-133, the smallest number)
    assert (got[:, :, 0] != 0)[plain[:, :, 0].abs() > 0.01].all() and torch.equal(got[:, :, 8], plain[:, :, 8])
    c["gate"][:, :, 3], c["gate"][:, :, 4] = -88.0, -1000.0
    assert (run(c)[:, :, 3:5].abs() <= 1.2e-38 * plain.abs().max()).all()
    c["gate"][:, :, 0], c["gate"][:, :, 1], c["gate"][:, :, 2] = -float("inf"), float("inf"), float("nan")
    c["v"][30, 0, 6] = float("inf")
    got = run(c)
    assert (got[:, :, 0] == 0).all() and torch.equal(got[:, :, 1], plain[:, :, 1]) and torch.isnan(got[:, :, 2]).all()
    assert (got[30:, :2, 6] == float("inf")).all()


def test_scores_of_minus_infinity_first(dev):
    """The first keys score -inf for every row: weight 0 once another key does not; alone, the formula's NaN."""
    c = inputs([100], 2, 1, 64, "bf16", 2, dev)
    c["q"][:, :, 0] = 1.0
    c["k"][:40, :, 0] = -float("inf")
    c["k"][40:, :, 0] = 0.0
    got = run(c)
    assert torch.isnan(got[:40]).all()
    # the same rows without those keys
    x = dict(c, q=c["q"][40:], k=c["k"][40:], v=c["v"][40:], cu=torch.tensor([0, 60], dtype=torch.int32, device=dev),
             lens=[60])
    check(x, got[40:], "behind 40 keys of -inf")


@pytest.mark.parametrize("amp", [0.0, 30.0])
def test_flat_and_extreme_scores(dev, amp):
    """All scores equal, and scores of hundreds that leave one key."""
    c = inputs([200, 65], 4, 2, 128, "bf16", 8, dev, amp=amp)
    check(c, run(c), f"amp {amp}")


def test_rising_scores(dev):
    """Every key scores above the ones before: the running maximum moves at every tile."""
    for D, step in ((64, 0.02), (128, 0.5), (256, 3.0)):
        c = inputs([600], 2, 2, D, "bf16", D, dev)
        c["q"][:] = 1.0
        c["k"][:] = (torch.arange(600, device=dev) * step / D * D ** 0.5)[:, None, None].to(torch.bfloat16)
        check(c, run(c), f"D {D} step {step}")


def test_offsets_out_of_range_are_clamped(dev):
    c = inputs([50, 30], 2, 1, 64, "bf16", 4, dev)
    want = run(c)
    y = dict(c, cu=torch.tensor([0, 50, 1 << 30], dtype=torch.int32, device=dev))
    assert torch.equal(run(y), want)
    y = dict(c, cu=torch.tensor([-7, 50, 80], dtype=torch.int32, device=dev))
    assert torch.equal(run(y), want)
    # offsets that go back: an empty sequence
    y = dict(c, cu=torch.tensor([0, 50, 20, 20], dtype=torch.int32, device=dev))
    got = run(y)
    assert torch.equal(got[:50], want[:50]) and (got[50:] == 7).all()


def test_no_rows(dev):
    c = inputs([5], 2, 1, 64, "bf16", 4, dev)
    empty = dict(c, cu=c["cu"][:1])
    assert (run(empty) == 7).all()
    none = {n: c[n][:0] if n in ("q", "k", "v") else c[n] for n in c}
    assert run(none).numel() == 0


def test_captured_and_replayed(dev):
    """One graph for a batch of 300 rows and up to 4 prompts, replayed over new lengths and values, eager calls between."""
    c = inputs([100, 200], 6, 2, 128, "bf16", 1, dev)
    c["cu"] = torch.tensor([0, 100, 300, 300, 300], dtype=torch.int32, device=dev)
    out = torch.zeros_like(c["q"])
    run(c, out)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        run(c, out)
    for i, lens in enumerate(([100, 200], [1, 1, 1, 297], [300], [40, 0, 64])):
        new = inputs(lens, 6, 2, 128, "bf16", 50 + i, dev, tail=300 - sum(lens))
        for n in ("q", "k", "v"):
            c[n].copy_(new[n])
        cu = offsets(lens)
        c["cu"].copy_(torch.from_numpy(np.concatenate([cu, np.full(5 - len(cu), cu[-1])]).astype(np.int32)))
        out.fill_(7.0)
        graph.replay()
        want = run(dict(c))
        torch.cuda.synchronize()
        assert torch.equal(out, want), lens
        check(dict(new, cu=c["cu"]), out, f"replay {lens}")


def test_two_streams_and_repeats(dev):
    """Calls on two streams at once, no workspace between them, and the same bits every time."""
    cases = [inputs([400, 90], 8, 2, 128, "bf16", 1, dev), inputs([33, 257], 8, 2, 256, "fp16", 2, dev, gate=True)]
    want = [run(c) for c in cases]
    outs = [torch.zeros_like(c["q"]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        for c, o, s in zip(cases, outs, streams):
            run(c, o, stream=s)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,Hq,Hkv", [([900], 4, 1), ([1500], 16, 4), ([250] * 8, 16, 4), ([2600], 8, 1),
                                         ([3, 1, 2] * 40, 3, 3)])
def test_every_shape_of_workgroup(dev, D, lens, Hq, Hkv):
    """Batches that are shared out among a workgroup's waves by keys, by both and by rows."""
    c = inputs(lens, Hq, Hkv, D, "bf16", D + len(lens), dev, gate=D == 256)
    check(c, run(c), f"D {D} {len(lens)} x {lens[0]} heads {Hq}/{Hkv}")


@pytest.mark.parametrize("lens,Hq,Hkv", [
    ([(37 * i) % 200 for i in range(200)], 32, 8), ([0] * 3 + [260] * 120, 16, 16), ([(53 * i) % 61 for i in range(256)], 64, 16),
    ([(53 * i) % 9 for i in range(5000)], 4, 2), ([0] * 300 + [700, 0, 1], 8, 2), ([(29 * i) % 97 for i in range(257)], 8, 1)])
def test_many_turns_and_many_sequences(dev, lens, Hq, Hkv):
    """Grids of many turns (tiles in bands of levels), and more sequences than a wave holds offsets of, empty ones among
    them."""
    check_fast(inputs(lens, Hq, Hkv, 256, "bf16", len(lens), dev, lead=5, tail=3))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_short_sequences(dev, D, dtype):
    """Gates, rows outside the sequences, and values that are not finite, where a wave has a tile for itself."""
    lens = [1 + 7 * i % 9 for i in range(600)]
    c = inputs(lens, 4, 2, D, dtype, 3 * D, dev, gate=True, lead=2, tail=2)
    got = run(c)
    check(c, got, f"D {D} {dtype}")
    assert (got[:2] == 7).all() and (got[-2:] == 7).all()
    y = dict(c, v=c["v"].clone())
    at = 2 + int(np.cumsum(lens)[299]) + 1  # the second row of a sequence of 4
    assert lens[300] == 4
    y["v"][at, 0, 3], y["v"][0], y["v"][-1] = float("nan"), float("nan"), float("inf")
    hit = run(y)
    same = torch.ones_like(got, dtype=torch.bool)
    same[at:at + 3, :2, 3] = False
    assert torch.equal(hit[same], got[same]) and torch.isnan(hit[at:at + 3, :2, 3]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scores_that_jump(dev, dtype):
    """A key now and then scores far above all before it, in tiles of any key group, for some rows only."""
    for D, n in ((64, 700), (128, 333), (256, 130)):
        c = inputs([n], 4, 1, D, dtype, n, dev, amp=0.3)
        c["q"][::3, :, 0] = 4.0
        c["k"][:, :, 0] = 0.0
        for i, at in enumerate(range(5, n, 41)):
            c["k"][at, :, 0] = 3.0 * D ** 0.5 * (i + 1) / 4  # 3 (i + 1) above the others in score
        check(c, run(c), f"{dtype} D {D}")


@pytest.mark.parametrize("which", ["q", "gate"])
def test_out_may_be_the_queries_or_the_gates(dev, which):
    for lens, D in (([100, 3], 64), ([300] * 9, 128), ([260], 256), ([200] * 30, 256)):
        c = inputs(lens, 8, 2, D, "bf16", D, dev, gate=True)
        want = run(c)
        assert torch.equal(run(c, c[which]), want)


def test_rows_past_2_gib(dev):
    """Rows 32 KiB apart: the last ones start behind 2^31 bytes of every operand."""
    T, H, D = 70000, 2, 64
    x = torch.zeros(T, 16384, device=dev, dtype=torch.bfloat16)
    part = lambda i: x[:, i * H * D:(i + 1) * H * D].view(T, H, D)
    g = torch.Generator(device=dev).manual_seed(1)
    for i in range(4):
        part(i).copy_(torch.randn(T, H, D, device=dev, generator=g))
    q, k, v, gate, out = (part(i) for i in range(5))
    # the rows in between belong to no sequence
    for cu in ([0, 1, 701], [69700, 70000]):
        pkv.attn_packed(q, k, v, torch.tensor(cu, dtype=torch.int32, device=dev), out, 0.125, gate=gate)
    for a, b in ((1, 701), (69700, 70000)):
        c = dict(q=q[a:b].contiguous(), k=k[a:b].contiguous(), v=v[a:b].contiguous(), gate=gate[a:b].contiguous(),
                 cu=torch.tensor([0, b - a], dtype=torch.int32, device=dev), lens=[b - a], lead=0, scale=0.125)
        check(c, out[a:b], f"rows {a}..{b}")
    assert (out[701:69700] == 0).all() and (x[:, 5 * H * D:] == 0).all()
