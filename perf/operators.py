"""Performance cases of the operators around a step's paged attention: the
step planned on the GPU, rotary positions, rotary rows, and attention over
whole prompts that are kept in no cache.

Kinds of case (`kind`), one pass each:
  packed     attention over a batch of whole prompts, packed rows of different lengths, causal, grouped heads;
             gated like the layer whose projection rows are [hq x (q | gate) | k | v], else rows [q | k | v]
  rope       q and k rows of a projection normed (or not) and rotated by positions on three axes
  positions  the time / height / width position of every row of a step, from the images and videos in the
             sequences (`media` of them each): of fresh prompts, or of one decode row a sequence
  plan       a step's block tables, slot map and row metadata from the requests' lengths, pages taken from a
             free list that lies on the GPU

`own` false: the same in elementary torch operations. Sequence lengths are
spread over their range (log-uniformly where that spans more than a factor of
ten) by `mix`; the seed picks the values.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE = 16
EPS = 1e-6
NO_BLOCKS, INVALID = 802, 1  # a row's status where its pages, or its lengths, do not allow it
MAX_FLOPS = 2.1e12           # of a drawn batch of prompts (the largest listed one: 2.2e12)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one short prompt to be embedded or scored: the smallest call, launch and latency
        dict(name="packed_one_short", kind="packed", hq=16, hkv=4, d=256, dtype="bf16", gate=True, batch=1, lo=37, hi=37,
             mix=1),
        # a step of fresh prompts of mixed lengths at the 16 / 4 layer
        dict(name="packed_10_mixed", kind="packed", hq=16, hkv=4, d=256, dtype="bf16", gate=True, batch=10, lo=37, hi=1900,
             mix=2),
        # documents to be scored at heads of 128 dims
        dict(name="packed_24_d128", kind="packed", hq=32, hkv=8, d=128, dtype="bf16", gate=False, batch=24, lo=60, hi=4096,
             mix=3),
        # one long document (the largest by flops)
        dict(name="packed_one_16k_d128", kind="packed", hq=32, hkv=8, d=128, dtype="bf16", gate=False, batch=1, lo=16384,
             hi=16384, mix=4),
        # many short passages through a small embedding model, fp16
        dict(name="packed_200_d64_fp16", kind="packed", hq=12, hkv=2, d=64, dtype="fp16", gate=False, batch=200, lo=1, hi=300,
             mix=5),
        # one prompt at 24 query heads
        dict(name="packed_one_4k_g6", kind="packed", hq=24, hkv=4, d=256, dtype="bf16", gate=True, batch=1, lo=4096, hi=4096,
             mix=6),
        # a decode step's rows, norm and partial rotation as the 16 / 4 layer has them
        dict(name="rope_64", kind="rope", hq=16, hkv=4, d=256, rot=64, dtype="bf16", gate=True, norm=True, adjacent=False,
             rows=64, mix=7),
        # a long prompt's rows, whole heads of 128 dims rotated
        dict(name="rope_16k_d128", kind="rope", hq=32, hkv=8, d=128, rot=128, dtype="bf16", gate=False, norm=False,
             adjacent=False, rows=16384, mix=8),
        # decode rows of conversations with a few images each
        dict(name="positions_64_decode", kind="positions", batch=64, lo=1, hi=1, media=5, video=False, mix=9),
        # long videos, a span for every few frames
        dict(name="positions_4_video", kind="positions", batch=4, lo=6000, hi=9000, media=600, video=True, mix=10),
        # a decode step over 64 running requests
        dict(name="plan_64_step", kind="plan", rows=64, lo=512, hi=8192, tlo=1, thi=1, free=4.0, mix=11),
        # a step of prompt chunks beside running requests
        dict(name="plan_300_chunks", kind="plan", rows=300, lo=1, hi=30000, tlo=1, thi=2000, free=1.5, mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _spread(rng, lo, hi):
    return _log(rng, lo, hi) if lo > 0 and hi > 10 * lo else rng.randint(lo, hi)


# (hq, hkv, d): the layers of the paged path, their heads sharded, and generic ones, odd groups among them
SHAPES = [(16, 4, 256), (24, 4, 256), (16, 2, 256), (4, 1, 256), (32, 8, 128), (8, 1, 128), (20, 4, 128), (7, 1, 128),
          (12, 2, 64), (14, 2, 64), (9, 3, 64), (16, 16, 64)]


def draw(rng):
    while True:
        kind = rng.choice(["packed", "packed", "packed", "packed", "rope", "rope", "positions", "plan"])
        case = dict(kind=kind, mix=rng.randrange(100, 1 << 20))
        if kind in ("packed", "rope"):
            hq, hkv, d = rng.choice(SHAPES)
            case.update(hq=hq, hkv=hkv, d=d, dtype=rng.choice(["bf16", "bf16", "fp16"]), gate=d == 256)
        if kind == "packed":
            case["batch"] = _log(rng, 1, 256)
            case["lo"] = _log(rng, 1, 8192)
            case["hi"] = min(16384, int(case["lo"] * rng.uniform(1.0, 40.0)))
            rows = sum(_lengths(case))
            if rows > 32768 or work(case)["flops"] > MAX_FLOPS:
                continue
        elif kind == "rope":
            case["rot"] = rng.choice([case["d"], case["d"], case["d"] // 4, 64])
            case["norm"], case["adjacent"] = rng.random() < 0.5, rng.random() < 0.3
            case["rows"] = _log(rng, 1, 16384)
            if case["rows"] * (case["hq"] + case["hkv"]) * case["d"] > 16384 * 40 * 128:
                continue
        elif kind == "positions":
            case["video"] = rng.random() < 0.5
            case["media"] = _log(rng, 1, 600)
            case["batch"] = _log(rng, 1, 128)
            case["lo"] = rng.choice([1, _log(rng, 1, 9000)])
            case["hi"] = case["lo"] if case["lo"] == 1 else min(9000, int(case["lo"] * rng.uniform(1.0, 5.0)))
            if case["batch"] * case["media"] > 4096 or sum(_lengths(case)) > 65536:
                continue
        else:
            case["rows"] = _log(rng, 1, 1500)
            case["lo"] = _log(rng, 1, 8192)
            case["hi"] = int(case["lo"] * rng.uniform(1.0, 16.0))
            case["tlo"] = rng.choice([1, 1, _log(rng, 1, 512)])
            case["thi"] = case["tlo"] if rng.random() < 0.4 else int(case["tlo"] * rng.uniform(1.0, 60.0)) + 1
            case["free"] = rng.choice([4.0, 1.5, 0.6])  # free pages over those asked for: below 1 some rows get none
            if case["rows"] * (case["hi"] + case["thi"]) > 16 << 20 or sum(abs(n) for n in _plan_lengths(case)[1]) > 65536:
                continue
        return case


def _lengths(case):
    rng = random.Random(case["mix"])
    return [_spread(rng, case["lo"], case["hi"]) for _ in range(case["batch"])]


def _plan_lengths(case):
    """Per row: positions cached, tokens this step feeds (0: none, below 0: padding rows), pages held."""
    rng = random.Random(case["mix"])
    ctx = [_spread(rng, case["lo"], case["hi"]) for _ in range(case["rows"])]
    new = [_spread(rng, case["tlo"], case["thi"]) for _ in ctx]
    if case["thi"] > 1:
        # most rows decode, some are idle; fresh prompts have nothing cached
        new = [n if i % 6 == 0 else (0 if i % 11 == 3 else 1) for i, n in enumerate(new)]
        ctx = [0 if i % 18 == 0 else c for i, c in enumerate(ctx)]
    for i in range(len(new) - len(new) // 16, len(new)):
        new[i] = -1  # the bucket's padding
    held = [-(-c // PAGE) + (1 if i % 9 == 4 else 0) for i, c in enumerate(ctx)]
    return ctx, new, held


def _plan_pages(case):
    ctx, new, held = _plan_lengths(case)
    return [max(0, -(-(c + n) // PAGE) - h) if n > 0 else 0 for c, n, h in zip(ctx, new, held)]


def work(case):
    if case["kind"] == "packed":
        lens, hq, hkv, d = _lengths(case), case["hq"], case["hkv"], case["d"]
        pairs = sum(n * (n + 1) // 2 for n in lens)
        rows = sum(lens)
        return {"bytes": rows * 2 * d * ((3 if case["gate"] else 2) * hq + 2 * hkv), "flops": 4 * d * hq * pairs}
    if case["kind"] == "rope":
        rows = case["rows"]
        return {"bytes": rows * (12 + 4 * (case["hq"] + case["hkv"]) * case["d"]), "flops": 0}
    if case["kind"] == "positions":
        # pos, row -> three positions; the spans
        return {"bytes": sum(_lengths(case)) * (8 + 12) + case["batch"] * case["media"] * 24, "flops": 0}
    new = _plan_lengths(case)[1]
    return {"bytes": sum(abs(n) for n in new) * 12 + case["rows"] * 36 + 8 * sum(_plan_pages(case)), "flops": 0}


# --------------------------------------------------------------------------
# inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * seed + 7)
    return g


def _dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype)).to(DEV)


def _projection(case, rows, g):
    """The projection rows, and the views of their q, gate (or None), k and v."""
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    wide = 2 if case["gate"] else 1
    x = torch.randn(rows, (wide * hq + 2 * hkv) * d, device=DEV, dtype=TYPES[case["dtype"]], generator=g)
    q = x[:, :wide * hq * d].view(rows, hq, wide, d)
    k = x[:, wide * hq * d:(wide * hq + hkv) * d].view(rows, hkv, d)
    v = x[:, (wide * hq + hkv) * d:].view(rows, hkv, d)
    return q[:, :, 0], q[:, :, 1] if case["gate"] else None, k, v


def _prepare_packed(case, seed):
    g, lens = _gen(seed), _lengths(case)
    rows, dt = sum(lens), TYPES[case["dtype"]]
    _, gate, _, v = _projection(case, rows, g)
    # q and k normed and rotated, rows of their own: scores of a few units' spread
    q = torch.randn(rows, case["hq"], case["d"], device=DEV, dtype=dt, generator=g).mul_(1.5)
    k = torch.randn(rows, case["hkv"], case["d"], device=DEV, dtype=dt, generator=g).mul_(1.5)
    return dict(case=case, lens=lens, q=q, k=k, v=v, gate=gate, cu=_dev(np.concatenate([[0], np.cumsum(lens)])),
                scale=case["d"] ** -0.5, out=torch.empty_like(q))


def _prepare_rope(case, seed):
    g, n, half = _gen(seed), case["rows"], case["rot"] // 2
    q, _, k, _ = _projection(case, n, g)
    rng = np.random.default_rng(1000003 * seed + 11)
    # text rows have one position on all axes, rows of images and videos three
    start = int(rng.integers(0, 250000))
    t = start + np.arange(n)
    image = (np.arange(n) // 50) % 2
    pos = np.stack([t, t + image * rng.integers(0, 40, n), t + image * rng.integers(0, 60, n)])
    if case["mix"] % 2:  # axes interleaved over the low frequencies' dims, else in sections
        axes = np.where(np.arange(half) < 3 * (half // 3), np.arange(half) % 3, 0)
    else:
        axes = np.repeat([0, 1, 2], [half - 2 * (3 * half // 8), 3 * half // 8, 3 * half // 8])
    st = dict(case=case, q=q, k=k, rope=_dev(pos), axes=_dev(axes),
              inv_freq=(1.0 / 1e7 ** (torch.arange(half, device=DEV, dtype=torch.float64) / half)).float(),
              q_out=torch.empty(q.shape, device=DEV, dtype=q.dtype), k_out=torch.empty(k.shape, device=DEV, dtype=k.dtype))
    if case["norm"]:
        st["q_norm"] = 1.5 + 0.2 * torch.randn(case["d"], device=DEV, generator=g)
        st["k_norm"] = 1.5 + 0.2 * torch.randn(case["d"], device=DEV, generator=g)
    return st


def _spans(case, seed):
    """Per request: starts and (time, height, width, step) of its media spans, text between them."""
    rng = np.random.default_rng(1000003 * seed + 13)
    n, m = case["batch"], case["media"]
    t = rng.integers(1, 4, (n, m)) if case["video"] else np.ones((n, m), np.int64)
    h, w = rng.integers(2, 14, (n, m)), rng.integers(2, 14, (n, m))
    step = rng.integers(1, 4, (n, m)) if case["video"] else np.ones((n, m), np.int64)
    gap = rng.integers(0, 12 if case["video"] else 200, (n, m))
    start = np.cumsum(gap + np.concatenate([np.zeros((n, 1), np.int64), (t * h * w)[:, :-1]], 1), 1)
    return np.stack([start, t, h, w, step], 2)


def _prepare_positions(case, seed):
    spans, lens = _spans(case, seed), _lengths(case)
    n, m = case["batch"], case["media"]
    if case["lo"] == 1 and case["hi"] == 1:
        # one decode row a sequence, behind or between its media
        rng = np.random.default_rng(1000003 * seed + 17)
        end = spans[:, -1, 0] + spans[:, -1, 1] * spans[:, -1, 2] * spans[:, -1, 3]
        pos, seq = end - 100 + rng.integers(0, 3000, n), np.arange(n)
        pos = np.maximum(pos, 0)
    else:
        pos = np.concatenate([np.arange(k) for k in lens])
        seq = np.repeat(np.arange(n), lens)
    return dict(case=case, fresh=not (case["lo"] == 1 and case["hi"] == 1), pos=_dev(pos), seq=_dev(seq),
                span_cu=_dev(np.arange(n + 1) * m), spans=_dev(spans.reshape(n * m, 5)),
                base=_dev(_bases(spans).reshape(-1)), rope=torch.zeros(3, len(pos), device=DEV, dtype=torch.int32))


def _bases(spans):
    """The position at which each span starts."""
    s, t, h, w, step = (spans[..., i].astype(np.int64) for i in range(5))
    gain = np.maximum(np.maximum((t - 1) * step + 1, h), w) - t * h * w
    return s + np.cumsum(gain, -1) - gain


def _plan_inputs(case, seed):
    ctx, new, held = _plan_lengths(case)
    rng = np.random.default_rng(1000003 * seed + 19)
    asked = sum(_plan_pages(case))
    free = int(case["free"] * asked) + (3 if case["free"] >= 1 else 0)
    ids = rng.permutation(sum(held) + free).astype(np.int32)
    width = max(max(held), -(-max(c + max(n, 0) for c, n in zip(ctx, new)) // PAGE)) + 2
    table = np.zeros((case["rows"], width), np.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = ids[at:at + h]
        at += h
    stack = np.zeros(len(ids), np.int32)  # the pages of the pool that are free, taken from the end
    stack[:free] = ids[at:]
    return np.array(ctx), np.array(new), np.array(held), table, stack, free


def _prepare_plan(case, seed):
    ctx, new, held, table, stack, free = _plan_inputs(case, seed)
    n, T = case["rows"], int(np.abs(new).sum()) + 5
    empty = lambda k: torch.zeros(k, device=DEV, dtype=torch.int32)
    return dict(case=case, T=T, pool=len(stack), len=_dev(ctx), held=_dev(held), ntok=_dev(new), table=_dev(table),
                free_list=_dev(stack), free_count=_dev([free]), pos=empty(T), slot_map=empty(T), tok_seq=empty(T),
                cu=empty(n + 1), limits=empty(n), len_out=empty(n), held_out=empty(n), free_out=empty(1),
                status=empty(n))


def prepare(case, seed):
    return {"packed": _prepare_packed, "rope": _prepare_rope, "positions": _prepare_positions,
            "plan": _prepare_plan}[case["kind"]](case, seed)


# --------------------------------------------------------------------------
# one pass: the framework's calls, or plain torch

def _pkv():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pocket-engine_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import pkv
    return pkv


def _own_packed(pkv, st):
    pkv.attn_packed(st["q"], st["k"], st["v"], st["cu"], st["out"], st["scale"], gate=st["gate"])
    return {"out": st["out"]}


def _own_rope(pkv, st):
    pkv.rope_rows(st["q"], st["k"], st["rope"], st["axes"], st["inv_freq"], st["q_out"], st["k_out"],
                  q_norm=st.get("q_norm"), k_norm=st.get("k_norm"), eps=EPS, adjacent=st["case"]["adjacent"])
    return {"q": st["q_out"], "k": st["k_out"]}


def _own_positions(pkv, st):
    if st["fresh"]:
        pkv.rope_spans(st["span_cu"], st["spans"], st["base"])
    pkv.rope_positions(st["pos"], st["seq"], st["span_cu"], st["spans"], st["base"], st["rope"])
    return {"rope": st["rope"], "base": st["base"]}


def _own_plan(pkv, st):
    pkv.plan_step(st["len"], st["held"], st["ntok"], st["table"], PAGE, st["pool"], st["pos"], st["slot_map"],
                  st["tok_seq"], st["cu"], st["limits"], st["len_out"], st["held_out"], st["status"],
                  free_list=st["free_list"], free_count=st["free_count"], free_count_out=st["free_out"])
    return {n: st[n] for n in ("table", "pos", "slot_map", "tok_seq", "cu", "limits", "len_out", "held_out", "free_out",
                               "status")}


def _attend(q, k, v, scale):
    """Causal softmax attention of [.., H, L, d] float32, in place where it can be."""
    n = q.shape[-2]
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(scale)
    at = torch.arange(n, device=q.device)
    s.masked_fill_(at[None] > at[:, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    return torch.matmul(s, v).div_(s.sum(-1, keepdim=True))


def _plain_packed(st):
    lens, hq, hkv = st["lens"], st["case"]["hq"], st["case"]["hkv"]
    B, top = len(lens), max(lens)
    heads = torch.arange(hq, device=DEV) // (hq // hkv)
    q, k, v = st["q"].float(), st["k"].float()[:, heads], st["v"].float()[:, heads]
    if B * top * top <= 3 * sum(n * n for n in lens) or B * top * top * hq <= 1 << 28:
        # the whole batch at once, short prompts filled up with the last row
        at = torch.arange(top, device=DEV)
        cu = st["cu"].long()
        inside = at[None] < (cu[1:] - cu[:-1])[:, None]
        idx = torch.minimum(cu[:-1, None] + at, cu[1:, None] - 1)
        x = _attend(*(y[idx].transpose(1, 2).contiguous() for y in (q, k, v)), st["scale"])
        out = x.transpose(1, 2)[inside]
    else:
        parts = (y.split(lens) for y in (q, k, v))
        out = torch.cat([_attend(*(y.transpose(0, 1).contiguous() for y in one), st["scale"]).transpose(0, 1)
                         for one in zip(*parts)])
    if st["gate"] is not None:
        out = out * torch.sigmoid(st["gate"].float())
    return {"out": out.to(st["q"].dtype)}


def _plain_rope(st):
    half, rot = st["case"]["rot"] // 2, st["case"]["rot"]
    ang = st["rope"][st["axes"].long()].double().t() * st["inv_freq"].double()
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]

    def rows(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
        if st["case"]["adjacent"]:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :half], y[..., half:rot]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)

    return {"q": rows(st["q"], st.get("q_norm")), "k": rows(st["k"], st.get("k_norm"))}


def _plain_positions(st):
    pos, seq, cu = st["pos"].long(), st["seq"].long(), st["span_cu"].long()
    start, t, h, w, step = st["spans"].long().t()
    base = st["base"].long()
    if st["fresh"]:
        gain = torch.maximum(torch.maximum((t - 1) * step + 1, h), w) - t * h * w
        before = gain.cumsum(0) - gain
        base = start + before - before[cu[:-1]].repeat_interleave(cu[1:] - cu[:-1], output_size=len(t))
    # the last span of the row's sequence that starts at or before it
    far = 1 << 32
    owner = torch.searchsorted(cu, torch.arange(len(t), device=DEV), right=True) - 1
    at = torch.searchsorted(owner * far + start, seq * far + pos, right=True) - 1
    has = at >= cu[seq]
    at = at.clamp(min=0)
    t, h, w, step, b = t[at], h[at], w[at], step[at], base[at]
    j = pos - start[at]
    inside = has & (j < t * h * w)
    after = torch.where(has, b + torch.maximum(torch.maximum((t - 1) * step + 1, h), w) + j - t * h * w, pos)
    rope = torch.stack([torch.where(inside, b + j // (h * w) * step, after),
                        torch.where(inside, b + j // w % h, after), torch.where(inside, b + j % w, after)])
    return {"rope": rope.int(), "base": base.int()}


def _plain_plan(st):
    T, table = st["T"], st["table"].long()
    length, held, ntok, free = (st[n].long() for n in ("len", "held", "ntok", "free_count"))
    rows, width = table.shape
    count = ntok.abs()
    incl = count.cumsum(0)
    fits = incl <= T
    total = torch.where(fits, incl, 0).amax()
    cu = torch.cat([incl.new_zeros(1), torch.where(fits, incl, total)])
    end = length + ntok
    live = (ntok > 0) & fits
    wrong = live & ((length < 0) | (held < 0) | (held > width) | (end > width * PAGE))
    need = torch.where(live & ~wrong, ((end + PAGE - 1) // PAGE - held).clamp(min=0), 0)
    asked = need.cumsum(0)
    given = (need == 0) | (asked <= free)
    good = live & ~wrong & given
    take = torch.where(good, need, 0)
    col = torch.arange(width, device=DEV)
    new = (col >= held[:, None]) & (col < (held + take)[:, None])
    src = (free - asked)[:, None] + col - held[:, None]
    table = torch.where(new, st["free_list"].long()[src.clamp(0, st["pool"] - 1)], table)
    held_out = held + take
    limits = torch.where((ntok >= 0) & (good | (ntok == 0)), held_out * PAGE - 1, -1)
    status = torch.where((count > 0) & ~fits | wrong, INVALID, torch.where(live & ~given, NO_BLOCKS, 0))
    t = torch.arange(T, device=DEV)
    row = torch.searchsorted(cu[1:], t, right=True).clamp(max=rows - 1)
    k = t - cu[row]
    pos = torch.where(good[row], length[row] + k, k)
    slot = torch.where(good[row], table[row, (pos // PAGE).clamp(0, width - 1)] * PAGE + pos % PAGE, -1)
    real = t < total
    out = dict(table=table, pos=torch.where(real, pos, 0), slot_map=torch.where(real, slot, -1),
               tok_seq=torch.where(real, row, 0), cu=cu, limits=limits,
               len_out=length + torch.where(good, ntok, 0), held_out=held_out,
               free_out=free - torch.where(given & (need > 0), asked, 0).amax(), status=status)
    return {n: x.int() for n, x in out.items()}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"packed": _own_packed, "rope": _own_rope, "positions": _own_positions,
                "plan": _own_plan}[kind](_pkv(), state)
    return {"packed": _plain_packed, "rope": _plain_rope, "positions": _plain_positions, "plan": _plain_plan}[kind](state)


# --------------------------------------------------------------------------
# the same from the definitions, in 64 bits and whole numbers

def _exact_packed(case, seed):
    st = _prepare_packed(case, seed)
    G = case["hq"] // case["hkv"]
    out = torch.empty(st["q"].shape, device=DEV, dtype=torch.float64)
    a = 0
    for n in st["lens"]:
        for h in range(case["hq"]):
            k, v = (st[x][a:a + n, h // G].double().contiguous() for x in ("k", "v"))
            kt = k.t().contiguous()
            for r in range(0, n, 4096):
                e = min(n, r + 4096)
                x = st["q"][a + r:a + e, h].double() @ kt[:, :e] * st["scale"]
                x = x + torch.full((e - r, e), -math.inf, device=DEV, dtype=torch.float64).triu_(r + 1)
                out[a + r:a + e, h] = torch.softmax(x, -1) @ v[:e]
        a += n
    if case["gate"]:
        out = out / (1 + torch.exp(-st["gate"].double()))
    return {"out": out}


def _exact_rope(case, seed):
    st = _prepare_rope(case, seed)
    rot = case["rot"]
    got = {}
    for n, w in (("q", st.get("q_norm")), ("k", st.get("k_norm"))):
        y = st[n].double()
        if w is not None:
            y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
        z = y.clone()
        for i in range(rot // 2):
            lo, hi = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + rot // 2)
            angle = st["rope"][int(st["axes"][i])].double() * float(st["inv_freq"][i])
            turn = torch.polar(torch.ones_like(angle), angle)[:, None]
            both = torch.complex(y[..., lo], y[..., hi]) * turn
            z[..., lo], z[..., hi] = both.real, both.imag
        got[n] = z
    return got


def _exact_positions(case, seed):
    st = _prepare_positions(case, seed)
    pos, seq, spans = st["pos"].cpu().numpy(), st["seq"].cpu().numpy(), _spans(case, seed)
    rope = np.zeros((3, len(pos)), np.int64)
    base = np.zeros(spans.shape[:2], np.int64)
    for s in range(case["batch"]):
        # walk the sequence: text and media in turn, each from where the last one ended
        mine = np.flatnonzero(seq == s)
        p, at, nxt = pos[mine], 0, 0
        for i, (start, t, h, w, step) in enumerate(spans[s].tolist() + [[1 << 30, 0, 0, 0, 0]]):
            text = (p >= at) & (p < start)
            rope[:, mine[text]] = nxt + p[text] - at
            nxt += start - at
            at = start + t * h * w
            here = (p >= start) & (p < at)
            if i < case["media"]:
                base[s, i] = nxt
                grid = np.indices((t, h, w)).reshape(3, -1)
                rope[:, mine[here]] = (nxt + grid * np.array([[step], [1], [1]]))[:, p[here] - start]
                nxt += max((t - 1) * step + 1, h, w)
    return {"rope": torch.from_numpy(rope).int(), "base": torch.from_numpy(base.reshape(-1)).int()}


def _exact_plan(case, seed):
    ctx, new, held, table, stack, free = _plan_inputs(case, seed)
    n, T = case["rows"], int(np.abs(new).sum()) + 5
    stack, width = stack[:free].tolist(), table.shape[1]
    pos, slot, seq, cu = np.zeros(T, int), np.full(T, -1), np.zeros(T, int), [0]
    limits, status, ctx, held, short = [], [], ctx.copy(), held.copy(), False
    for s in range(n):
        a, k = cu[-1], int(new[s])
        need = max(0, -(-(int(ctx[s]) + k) // PAGE) - int(held[s])) if k > 0 else 0
        ok = k > 0 and ctx[s] + k <= width * PAGE
        if ok and need:
            short = short or need > len(stack)
        refused = ok and need > 0 and short
        seq[a:a + abs(k)] = s
        pos[a:a + abs(k)] = np.arange(abs(k))
        if ok and not refused:
            if need:
                table[s, held[s]:held[s] + need] = stack[-need:]
                del stack[-need:]
            p = ctx[s] + np.arange(k)
            pos[a:a + k], slot[a:a + k] = p, table[s, p // PAGE] * PAGE + p % PAGE
            ctx[s] += k
            held[s] += need
        limits.append(held[s] * PAGE - 1 if k == 0 or (ok and not refused) else -1)
        status.append(NO_BLOCKS if refused else INVALID if k > 0 and not ok else 0)
        cu.append(a + abs(k))
    got = dict(table=table, pos=pos, slot_map=slot, tok_seq=seq, cu=cu, limits=limits, len_out=ctx, held_out=held,
               free_out=[len(stack)], status=status)
    return {k: torch.from_numpy(np.array(x, np.int32)) for k, x in got.items()}


def exact(case, seed):
    return {"packed": _exact_packed, "rope": _exact_rope, "positions": _exact_positions,
            "plan": _exact_plan}[case["kind"]](case, seed)
