"""Rotary positions on three axes and rows rotated by them, on the GPU:
positions and span starts equal to a walk over the sequence, rows within their
rounding of the formula in 64 bits.

Bound of a row's element, u half a step of the type: the norm's factor and the
products in f32 are off by at most 2^-20 of |y_a| + |y_b| (a sum of D squares
below D 2^-24 of it, halved by the root: 2^-17 at 256 dims before the root's
half: taken as (D / 2 + 16) 2^-24), the angle's cos and sin by 2^-21, then u |out|, and below the type's smallest
normal number (2^-14 in fp16), where the spacing stays that number's, u times it (2^-25)."""
import numpy as np
import pytest
import torch

import pkv

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def walk(spans, n):
    """Positions of the first n tokens of a sequence, token by token, and where each span starts."""
    out, base, nxt = np.zeros((3, n), np.int64), [], 0
    at = 0
    spans = [tuple(int(x) for x in s) for s in spans]
    for start, t, h, w, step in spans + [(1 << 40, 1, 1, 1, 1)]:
        if t < 1 or h < 1 or w < 1 or step < 0:
            base.append(nxt + start - at)  # text: nothing moves
            continue
        m = min(start, n)
        if m > at:
            out[:, at:m] = nxt + np.arange(m - at)
        nxt += start - at
        at = start
        base.append(nxt)
        if start >= 1 << 40:
            break
        for i in range(t):
            for j in range(h):
                for k in range(w):
                    if at < n:
                        out[:, at] = nxt + i * step, nxt + j, nxt + k
                    at += 1
        nxt += max((t - 1) * step + 1, h, w)
    return out, base[:len(spans)]


def batch(reqs, dev):
    cu = np.concatenate([[0], np.cumsum([len(r) for r in reqs])])
    flat = np.array([s for r in reqs for s in r], np.int32).reshape(-1, 5)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)
    return i32(cu), i32(flat), torch.full((len(flat),), -5, dtype=torch.int32, device=dev)


def random_spans(rng, m, video=True):
    out, at = [], 0
    for _ in range(m):
        at += int(rng.integers(0, 9))
        t, h, w, step = int(rng.integers(1, 4)) if video else 1, int(rng.integers(1, 7)), int(rng.integers(1, 7)), int(
            rng.integers(0, 4))
        out.append((at, t, h, w, step))
        at += t * h * w
    return out


REQS = [[], [(0, 1, 1, 1, 1)], [(3, 1, 4, 6, 1)], [(0, 3, 2, 2, 2), (12, 1, 5, 1, 1)], [(5, 2, 1, 1, 0), (7, 1, 1, 9, 0)]]


@pytest.mark.parametrize("many", [0, 1, 64, 65, 300, 1000])
def test_positions_match_a_walk(dev, many):
    rng = np.random.default_rng(many)
    reqs = REQS + [random_spans(rng, many)] + [random_spans(rng, k) for k in (7, 1)]
    cu, spans, base = batch(reqs, dev)
    pkv.rope_spans(cu, spans, base)
    pos, seq, want, starts = [], [], [], []
    for s, r in enumerate(reqs):
        n = (r[-1][0] + r[-1][1] * r[-1][2] * r[-1][3] if r else 0) + 40
        w, b = walk(r, n)
        starts += b
        pos.append(np.arange(n))
        seq.append(np.full(n, s))
        want.append(w)
    pos, seq, want = np.concatenate(pos), np.concatenate(seq), np.concatenate(want, 1)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)
    assert base.tolist() == starts
    rope = torch.full((3, len(pos) + 3), -1, dtype=torch.int32, device=dev)
    pkv.rope_positions(i32(pos), i32(seq), cu, spans, base, rope)
    assert np.array_equal(rope.cpu().numpy()[:, :-3], want) and (rope[:, -3:] == -1).all()
    # rows in any order: a decode step's, a shuffled one's
    order = rng.permutation(len(pos))
    pkv.rope_positions(i32(pos[order]), i32(seq[order]), cu, spans, base, rope)
    assert np.array_equal(rope.cpu().numpy()[:, :-3], want[:, order])


def test_rows_without_request_spans_or_sizes(dev):
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)
    # requests out of range and without spans: the position itself; a span of no size is text
    bad = [(2, 0, 4, 4, 1), (4, 1, -3, 2, 1), (6, 1, 2, 2, -1), (8, 1 << 20, 1 << 20, 1, 1), (10, 1, 2, 3, 1)]
    cu, spans, base = batch([bad, []], dev)
    pkv.rope_spans(cu, spans, base)
    assert base.tolist() == [2, 4, 6, 8, 10]
    pos, seq = i32([5, 9, 11, 16, 20, 3, 1 << 30, 4]), i32([0, 0, 0, 0, 0, 1, -1, 2])
    rope = torch.zeros(3, 8, dtype=torch.int32, device=dev)
    pkv.rope_positions(pos, seq, cu, spans, base, rope)
    assert rope.t().tolist() == [[5] * 3, [9] * 3, [10, 10, 11], [13] * 3, [17] * 3, [3] * 3, [1 << 30] * 3, [4] * 3]
    # no spans at all, no rows at all
    none = torch.zeros(0, 5, dtype=torch.int32, device=dev)
    pkv.rope_spans(i32([0, 0]), none, i32([]))
    pkv.rope_positions(pos, seq, i32([0, 0]), none, i32([]), rope)
    assert (rope == pos).all()
    pkv.rope_positions(i32([]), i32([]), cu, spans, base, rope)


def rows_case(T, Hq, Hkv, D, rot, dtype, norm, seed, dev, far=250000):
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    r = lambda H: (torch.randn(T, H, D, device=dev, generator=g) * 2).to(TYPES[dtype])
    half = rot // 2
    w = lambda: 1 + 0.3 * torch.randn(D, device=dev, generator=g)
    return dict(q=r(Hq), k=r(Hkv), rope=torch.from_numpy(rng.integers(0, far, (3, T + 2)).astype(np.int32)).to(dev),
                axes=torch.from_numpy(rng.integers(-1, 4, half).astype(np.int32)).to(dev),
                inv_freq=(1.0 / 1e6 ** (torch.arange(half, device=dev) / max(half, 1))).float(),
                q_norm=w() if norm else None, k_norm=w() if norm else None, D=D, rot=rot)


def want_rows(c, x, w, adjacent):
    D, half = c["D"], c["rot"] // 2
    T = x.shape[0]
    u = torch.finfo(x.dtype).eps / 2
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    axes = torch.where((c["axes"] == 1) | (c["axes"] == 2), c["axes"], 0).long()
    ang = (c["rope"][axes, :T].double().t() * c["inv_freq"].double())[:, None]
    a, b = (y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if adjacent else (y[..., :half], y[..., half:2 * half])
    lo, hi = a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()
    out, size = y.clone(), y.abs()
    if adjacent:
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = lo, hi
        size[..., 0:2 * half:2] = size[..., 1:2 * half:2] = a.abs() + b.abs()
    else:
        out[..., :half], out[..., half:2 * half] = lo, hi
        size[..., :half] = size[..., half:2 * half] = a.abs() + b.abs()
    return out, u * out.abs() + ((D / 2 + 16) * 2.0 ** -24 + 2.0 ** -21) * size + torch.finfo(x.dtype).tiny * u


def rows_check(c, adjacent=False, in_place=False):
    q, k = c["q"].clone(), c["k"].clone()
    qo, ko = (q, k) if in_place else (torch.full_like(q, 9), torch.full_like(k, 9))
    pkv.rope_rows(q, k, c["rope"], c["axes"], c["inv_freq"], qo, ko, q_norm=c["q_norm"], k_norm=c["k_norm"],
                  adjacent=adjacent)
    for n, got in (("q", qo), ("k", ko)):
        want, tol = want_rows(c, c[n], c[n + "_norm"], adjacent)
        err = (got.double() - want).abs()
        print(n, "worst over bound", float((err / tol).max()) if err.numel() else 0, flush=True)
        assert (err <= tol).all()
    return qo, ko


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 16), (128, 128), (128, 96), (128, 32), (256, 64), (256, 256), (256, 0)])
def test_rows_match_the_formula(dev, D, rot, adjacent, dtype):
    for T, Hq, Hkv in ((1, 4, 1), (3, 7, 3), (130, 16, 2)):
        for norm in (False, True):
            print("case", D, rot, adjacent, dtype, T, Hq, Hkv, norm, flush=True)
            c = rows_case(T, Hq, Hkv, D, rot, dtype, norm, T + D + rot, dev)
            a = rows_check(c, adjacent)
            b = rows_check(c, adjacent, in_place=True)
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_far_positions_and_one_norm(dev):
    c = rows_case(40, 4, 2, 128, 128, "fp16", True, 3, dev, far=(1 << 31) - 1)
    c["k_norm"] = None
    rows_check(c)
    c["rope"][:, ::2] *= -1  # positions below 0 turn the other way
    rows_check(c)


def test_strided_rows_and_values_left_alone(dev):
    """Views of a projection row, out inside wider rows; infinities stay in their pair."""
    T, Hq, Hkv, D = 33, 4, 2, 128
    c = rows_case(T, Hq, Hkv, D, 64, "bf16", False, 6, dev)
    want_q, want_k = rows_check(c)
    x = torch.zeros(T, (2 * Hq + 2 * Hkv) * D, device=dev, dtype=torch.bfloat16)
    q = x[:, :2 * Hq * D].view(T, Hq, 2, D)[:, :, 0]
    k = x[:, 2 * Hq * D:(2 * Hq + Hkv) * D].view(T, Hkv, D)
    q.copy_(c["q"])
    k.copy_(c["k"])
    wide = torch.full((T, Hq + Hkv + 1, D), 9.0, device=dev, dtype=torch.bfloat16)
    pkv.rope_rows(q, k, c["rope"], c["axes"], c["inv_freq"], wide[:, :Hq], wide[:, Hq:Hq + Hkv])
    assert torch.equal(wide[:, :Hq], want_q) and torch.equal(wide[:, Hq:Hq + Hkv], want_k) and (wide[:, -1] == 9).all()
    c["q"][5, 1, 100] = float("inf")
    c["q"][6, 1, 3] = float("nan")
    qo, ko = torch.empty_like(c["q"]), torch.empty_like(c["k"])
    pkv.rope_rows(c["q"], c["k"], c["rope"], c["axes"], c["inv_freq"], qo, ko)
    hit = torch.zeros_like(qo, dtype=torch.bool)
    hit[5, 1, 100] = hit[6, 1, 3] = hit[6, 1, 35] = True
    assert torch.equal(qo[~hit], want_q[~hit]) and qo[5, 1, 100] == float("inf") and torch.isnan(qo[6, 1, [3, 35]]).all()


def test_no_heads_and_replay(dev):
    c = rows_case(20, 4, 2, 64, 32, "bf16", True, 9, dev)
    wq, wk = rows_check(c)
    qo, ko = torch.zeros_like(c["q"]), torch.zeros_like(c["k"])
    args = (c["rope"], c["axes"], c["inv_freq"])
    pkv.rope_rows(c["q"], c["k"][:, :0], *args, qo, ko[:, :0], q_norm=c["q_norm"], k_norm=c["k_norm"])
    assert torch.equal(qo, wq) and (ko == 0).all()
    pkv.rope_rows(c["q"][:0], c["k"][:0], *args, qo[:0], ko[:0])
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        pkv.rope_rows(c["q"], c["k"], *args, qo, ko, q_norm=c["q_norm"], k_norm=c["k_norm"])
    for i in range(3):
        c["q"].mul_(1.5)
        c["rope"].add_(1000)
        graph.replay()
        w = rows_check(c)
        torch.cuda.synchronize()
        assert torch.equal(qo, w[0]) and torch.equal(ko, w[1])


@pytest.mark.parametrize("T,Hq,Hkv,D", [(17000, 32, 8, 128), (9000, 2, 1, 64), (5000, 16, 4, 256)])
def test_many_rows_are_the_same_rows(dev, T, Hq, Hkv, D):
    """Several tokens to a workgroup and outputs past the caches: bit for bit what short calls give, also at an odd end."""
    g = torch.Generator(device=dev).manual_seed(T)
    q, k = (torch.randn(T, h, D, device=dev, generator=g).bfloat16() for h in (Hq, Hkv))
    rope = torch.randint(0, 100000, (3, T), device=dev, generator=g, dtype=torch.int32)
    axes = torch.arange(D // 2, device=dev, dtype=torch.int32) % 3
    inv = (1e6 ** (-torch.arange(D // 2, device=dev) / (D // 2))).float()
    w = 1 + 0.1 * torch.randn(D, device=dev, generator=g)
    qo, ko = torch.full_like(q, 9), torch.full_like(k, 9)
    pkv.rope_rows(q, k, rope, axes, inv, qo, ko, q_norm=w)
    for a, b in ((0, 700), (T // 2, T // 2 + 333), (T - 411, T)):
        sq, sk = torch.zeros_like(q[a:b]), torch.zeros_like(k[a:b])
        pkv.rope_rows(q[a:b], k[a:b], rope[:, a:b].contiguous(), axes, inv, sq, sk, q_norm=w)
        assert torch.equal(qo[a:b], sq) and torch.equal(ko[a:b], sk)
    assert not (qo == 9).all(-1).any() and not (ko == 9).all(-1).any()
