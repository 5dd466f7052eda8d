"""Steps planned on the GPU (pkv.plan_step, pkv.plan_truncate) against a walk
over the rows and against the host manager, and a run of the operators around
a step together."""
import numpy as np
import pytest
import torch

import pkv

pytestmark = pytest.mark.gpu
SENT = -77


def walk(ctx, held, ntok, table, bs, pool, stack, T):
    """The step row by row: a list of free ids, popped from its end."""
    n, width = table.shape
    table, stack = table.copy(), None if stack is None else list(stack)
    pos, slot, seq = np.zeros(T, np.int64), np.full(T, -1), np.zeros(T, np.int64)
    cu, limits, status, ctx, held = [0], [], [], list(map(int, ctx)), list(map(int, held))
    short = full = False
    for s in range(n):
        a, k = cu[-1], int(ntok[s])
        full = full or (k != 0 and a + abs(k) > T)
        if full and k != 0:
            cu.append(a)
            status.append(1)
            limits.append(-1)
            continue
        wrong = k > 0 and (ctx[s] < 0 or held[s] < 0 or held[s] > width or ctx[s] + k > width * bs)
        need = max(0, -(-(ctx[s] + k) // bs) - held[s]) if k > 0 and not wrong else 0
        if need and (stack is None or need > len(stack)):
            short = True
        ok = k > 0 and not wrong and not (need and short)
        seq[a:a + abs(k)] = s
        pos[a:a + abs(k)] = np.arange(abs(k))
        if ok:
            if need:
                table[s, held[s]:held[s] + need] = stack[-need:]
                del stack[-need:]
            p = ctx[s] + np.arange(k)
            ids = table[s, p // bs]
            pos[a:a + k] = p
            slot[a:a + k] = np.where((ids >= 0) & (ids < pool), ids * bs + p % bs, -1)
            ctx[s] += k
            held[s] += need
        status.append(0 if ok or k <= 0 else 1 if wrong or stack is None else 802)
        limits.append(held[s] * bs - 1 if ok or k == 0 else -1)
        cu.append(a + abs(k))
    return dict(pos=pos, slot_map=slot, tok_seq=seq, cu=cu, limits=limits, status=status, len_out=ctx, held_out=held,
                table=table, free_count_out=None if stack is None else [len(stack)])


def i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)


def call(ctx, held, ntok, table, bs, pool, stack, T, dev, in_place=False, stream=None):
    n = len(ctx)
    new = lambda k: torch.full((k,), SENT, dtype=torch.int32, device=dev)
    a = dict(len=i32(ctx, dev), held=i32(held, dev), ntok=i32(ntok, dev), block_table=i32(table, dev))
    o = dict(pos=new(T), slot_map=new(T), tok_seq=new(T), cu=new(n + 1), limits=new(n), status=new(n))
    o["len_out"], o["held_out"] = (a["len"], a["held"]) if in_place else (new(n), new(n))
    f = {}
    if stack is not None:
        f["free_list"] = i32(list(stack) + [0] * (pool - len(stack)), dev)
        f["free_count"] = i32([len(stack)], dev)
        f["free_count_out"] = f["free_count"] if in_place else new(1)
    pkv.plan_step(block_size=bs, num_blocks=pool, stream=stream, **a, **o, **f)
    got = {k: v.cpu().numpy() for k, v in o.items()}
    got["table"] = a["block_table"].cpu().numpy()
    if stack is not None:
        got["free_count_out"] = f["free_count_out"].cpu().numpy()
    return got


def same(got, want):
    for k, w in want.items():
        if w is not None:
            assert np.array_equal(got[k], np.array(w)), (k, got[k], w)


def state(rng, n, bs, hi, extra, free, width=None):
    ctx = rng.integers(0, hi, n)
    ctx[::5] = 0
    held = -(-ctx // bs) + rng.integers(0, extra + 1, n)
    width = width or int(held.max() if n else 0) + 40
    ids = rng.permutation(int(held.sum()) + free)
    table, at = np.full((n, width), -3, np.int64), 0
    for s in range(n):
        table[s, :held[s]] = ids[at:at + held[s]]
        at += held[s]
    return ctx, held, table, ids[at:], len(ids)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,bs,most", [(1, 16, 1), (5, 16, 40), (64, 16, 1), (300, 16, 90), (1023, 1, 5), (1024, 16, 3),
                                       (1025, 64, 20), (2500, 16, 30)])
def test_steps_match_a_walk(dev, n, bs, most, in_place):
    rng = np.random.default_rng(n + bs)
    for free in (0, n // 2, 4 * n + most * n // bs + 10):
        print("case", n, bs, most, free, in_place, flush=True)
        ctx, held, table, stack, pool = state(rng, n, bs, 300, 2, free)
        pool = max(pool, 1)
        ntok = rng.integers(1, most + 1, n)
        ntok[rng.random(n) < 0.2] = 0
        ntok[rng.random(n) < 0.1] *= -1
        total = int(np.abs(ntok).sum())
        for T in {total, total + 37, max(1, total * 2 // 3)}:
            got = call(ctx, held, ntok, table, bs, pool, stack, T, dev, in_place)
            same(got, walk(ctx, held, ntok, table, bs, pool, stack, T))


def test_rows_that_do_not_fit_their_table(dev):
    # too long, negative lengths, more pages than the table has: those rows alone are refused
    ctx, held = [10, 60, -1, 5, 5, 70, 2], [1, 4, 0, -2, 9, 5, 1]
    ntok = [5, 5, 3, 2, 2, 11, 20]
    table = np.arange(35).reshape(7, 5)
    got = call(ctx, held, ntok, table, 16, 64, list(range(40, 60)), 60, dev)
    want = walk(ctx, held, ntok, table, 16, 64, list(range(40, 60)), 60)
    same(got, want)
    assert got["status"].tolist() == [0, 0, 1, 1, 1, 1, 0]
    # lengths that pass 31 bits
    big = (1 << 31) - 1
    got = call([big, 3, big], [1, 1, 1], [big, 1, -big], np.zeros((3, 4)), 16, 8, [1, 2], 10, dev)
    assert got["status"].tolist() == [1, 1, 1] and got["cu"].tolist() == [0] * 4 and (got["slot_map"] == -1).all()
    got = call([big, 3], [1, 1], [5, 1], np.zeros((2, 4)), 16, 8, [1, 2], 10, dev)
    assert got["status"].tolist() == [1, 0] and got["slot_map"].tolist()[:6] == [-1] * 5 + [3]
    got = call([3, 3], [1, 1], [-(1 << 31), 1], np.zeros((2, 4)), 16, 8, [1, 2], 10, dev)
    assert got["status"].tolist() == [1, 1]


def test_tables_as_they_are(dev):
    """Without a free list: only slots, a row that outgrows its pages is refused; ids outside the pool have no slot."""
    ctx, held, ntok = [10, 31, 3, 32], [1, 2, 1, 2], [3, 3, 2, 1]
    table = np.array([[4, 0, 0], [1, 2, 0], [99, 0, 0], [5, -1, 7]])
    got = call(ctx, held, ntok, table, 16, 8, None, 12, dev)
    same(got, walk(ctx, held, ntok, table, 16, 8, None, 12))
    assert got["status"].tolist() == [0, 1, 0, 1]
    assert got["slot_map"].tolist()[:3] == [74, 75, 76] and got["slot_map"].tolist()[6:8] == [-1, -1]


def test_no_rows_and_no_tokens(dev):
    got = call([], [], [], np.zeros((0, 4)), 16, 8, [1, 2, 3], 6, dev)
    assert got["cu"].tolist() == [0] and got["free_count_out"].tolist() == [3] and (got["slot_map"] == -1).all()
    got = call([5, 6], [1, 1], [0, 0], np.zeros((2, 4)), 16, 8, [1, 2, 3], 0, dev)
    assert got["cu"].tolist() == [0, 0, 0] and got["limits"].tolist() == [15, 15]
    got = call([5, 6], [1, 1], [0, 0], np.zeros((2, 4)), 16, 8, [1, 2, 3], 5000, dev)
    assert got["cu"].tolist() == [0, 0, 0] and (got["slot_map"] == -1).all() and (got["pos"] == 0).all()


def test_counts_outside_the_pool(dev):
    """A free count the pool cannot have is taken as its bounds."""
    for count in (-5, 1 << 30):
        a = dict(len=i32([0], dev), held=i32([0], dev), ntok=i32([3], dev), block_table=i32(np.zeros((1, 4)), dev))
        new = lambda k: torch.full((k,), SENT, dtype=torch.int32, device=dev)
        out = new(1)
        status = new(1)
        pkv.plan_step(**a, block_size=16, num_blocks=8, pos=new(3), slot_map=new(3), tok_seq=new(3), cu=new(2),
                      limits=new(1), len_out=new(1), held_out=new(1), status=status, free_list=i32(np.arange(8), dev),
                      free_count=i32([count], dev), free_count_out=out)
        assert status.tolist() == ([802] if count < 0 else [0]) and out.tolist() == ([0] if count < 0 else [7])
        assert a["block_table"][0, 0].item() == (0 if count < 0 else 7)


@pytest.mark.parametrize("n,bs", [(1, 16), (40, 16), (1500, 4)])
def test_truncate_gives_pages_back(dev, n, bs):
    rng = np.random.default_rng(n)
    ctx, held, table, stack, pool = state(rng, n, bs, 200, 3, 20)
    want_len = rng.integers(-3, 220, n)
    want_len[::4] = 0
    stack2, ctx2, held2 = list(stack), ctx.copy(), held.copy()
    for s in range(n):
        if 0 <= want_len[s] <= ctx[s]:
            keep = min(held[s], -(-want_len[s] // bs))
            stack2 += table[s, keep:held[s]].tolist()
            ctx2[s], held2[s] = want_len[s], keep
    l, h, t = i32(ctx, dev), i32(held, dev), i32(table, dev)
    f, c = i32(list(stack) + [-9] * (pool - len(stack)), dev), i32([len(stack)], dev)
    pkv.plan_truncate(i32(want_len, dev), l, h, t, bs, pool, f, c)
    assert np.array_equal(l.cpu(), ctx2) and np.array_equal(h.cpu(), held2) and np.array_equal(t.cpu(), table)
    assert c.item() == len(stack2) and f.tolist()[:len(stack2)] == stack2
    assert f.tolist()[len(stack2):] == [-9] * (pool - len(stack2))


def test_truncate_keeps_inside_the_list(dev):
    """More pages than the pool has room for (a state that no plan leaves): the list ends at the pool's size."""
    l, h, t = i32([64, 64], dev), i32([4, 4], dev), i32(np.arange(8).reshape(2, 4), dev)
    f, c = torch.full((12,), -9, dtype=torch.int32, device=dev), i32([5], dev)
    pkv.plan_truncate(i32([0, 0], dev), l, h, t, 16, 10, f, c)
    assert c.item() == 10 and f.tolist() == [-9] * 5 + [0, 1, 2, 3, 4] + [-9] * 2


def test_the_host_manager_hands_out_the_same_pages(dev):
    """A pool on the GPU and the host manager, fed the same steps: the same tables, slots and metadata, pages back too."""
    n, bs, pool, width, T = 6, 16, 200, 40, 128
    kv = pkv.Kv(pool)
    seqs = [kv.new_seq() for _ in range(n)]
    free = i32(np.arange(pool)[::-1], dev)  # the manager's list
    count, table = i32([pool], dev), i32(np.zeros((n, width)), dev)
    length, held = i32([0] * n, dev), i32([0] * n, dev)
    new = lambda k: torch.zeros(k, dtype=torch.int32, device=dev)
    pos, slot, seq, cu, limits, status = new(T), new(T), new(T), new(n + 1), new(n), new(n)
    rng = np.random.default_rng(5)
    lens = [0] * n
    for step in range(40):
        ntok = rng.integers(0, 20, n).tolist()
        if step % 7 == 6:  # rows end or are cut back
            cut = [int(rng.integers(0, lens[s] + 1)) if s % 2 == step % 2 else -1 for s in range(n)]
            for s, c in enumerate(cut):
                if c >= 0:
                    kv.truncate(seqs[s], c, True)
                    lens[s] = c
            pkv.plan_truncate(i32(cut, dev), length, held, table, bs, pool, free, count)
        for s in range(n):
            kv.reserve(seqs[s], lens[s] + ntok[s])
        want = kv.fill([(seqs[s], ntok[s]) for s in range(n)], T, width)
        pkv.plan_step(length, held, i32(ntok, dev), table, bs, pool, pos, slot, seq, cu, limits, length, held, status,
                      free_list=free, free_count=count, free_count_out=count)
        k = sum(ntok)
        for s in range(n):
            lens[s] += ntok[s]
            kv.set_len(seqs[s], lens[s])
        assert not status.any() and np.array_equal(cu.cpu(), want["cu"]) and np.array_equal(limits.cpu(), want["limits"])
        for a, name in ((pos, "pos"), (slot, "slot_map"), (seq, "tok_seq")):
            assert np.array_equal(a.cpu()[:k], want[name][:k]), name
        for s in range(n):
            assert table[s, :held[s]].tolist() == kv.blocks(seqs[s])
        assert count.item() == kv.free_count() and length.tolist() == lens


def test_a_captured_step_advances(dev):
    """A decode step captured once, replayed: every replay feeds the next token, pages taken as rows cross into them."""
    n, bs, width = 70, 16, 12
    rng = np.random.default_rng(8)
    ctx, held, table, stack, pool = state(rng, n, bs, 60, 0, 300, width)
    ntok = np.ones(n, np.int64)
    ntok[60:] = -1
    t = dict(len=i32(ctx, dev), held=i32(held, dev), ntok=i32(ntok, dev), block_table=i32(table, dev))
    new = lambda k: torch.zeros(k, dtype=torch.int32, device=dev)
    o = dict(pos=new(n), slot_map=new(n), tok_seq=new(n), cu=new(n + 1), limits=new(n), status=new(n))
    free, count = i32(list(stack) + [0] * (pool - len(stack)), dev), i32([len(stack)], dev)
    step = lambda: pkv.plan_step(**t, **o, block_size=bs, num_blocks=pool, len_out=t["len"], held_out=t["held"],
                                 free_list=free, free_count=count, free_count_out=count)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(40):
        want = walk(ctx, held, ntok, table, bs, pool, stack, n)
        if i % 10 == 9:
            step()  # an eager step between replays
        else:
            graph.replay()
        torch.cuda.synchronize()
        same({**{k: v.cpu().numpy() for k, v in o.items()}, "table": t["block_table"].cpu().numpy(),
              "len_out": t["len"].cpu().numpy(), "held_out": t["held"].cpu().numpy(),
              "free_count_out": count.cpu().numpy()}, want)
        ctx, held, table = np.array(want["len_out"]), np.array(want["held_out"]), want["table"]
        stack = stack[:want["free_count_out"][0]]


def test_the_operators_together(dev):
    """A step of fresh prompts with images: planned on the GPU, positions from the images' grids, rows normed and
    rotated, kept in the cache and attended through its pages (pkv_attn_prefill) and, from the rows themselves, as
    packed prompts (pkv_attn_packed); then a decode step behind them. Both attentions within bf16's rounding of each
    other: P rounded in both (2^-8 of sum w |v| each), q scaled and rounded in the paged one (2^-8 of a score of up to
    8: 2^-5 of sum w |v|), outputs rounded twice and once, so 2^-4 max |v| in all."""
    Hq, Hkv, D, bs, pool, width = 8, 2, 256, 16, 64, 24
    lens = [70, 1, 200, 33]
    T, n = sum(lens), len(lens)
    g = torch.Generator(device=dev).manual_seed(4)
    new = lambda *k: torch.zeros(*k, dtype=torch.int32, device=dev)
    length, held, count = new(n), new(n), i32([pool], dev)
    free, table = i32(np.random.default_rng(1).permutation(pool), dev), new(n, width)
    pos, slot, seq, cu, limits, status = new(T), new(T), new(T), new(n + 1), new(n), new(n)
    pkv.plan_step(length, held, i32(lens, dev), table, bs, pool, pos, slot, seq, cu, limits, length, held, status,
                  free_list=free, free_count=count, free_count_out=count)
    reqs = [[(4, 1, 5, 7, 1)], [], [(0, 3, 4, 4, 2), (60, 1, 8, 8, 1)], [(30, 1, 9, 9, 1)]]
    scu = i32(np.concatenate([[0], np.cumsum([len(r) for r in reqs])]), dev)
    spans = i32(np.array([s for r in reqs for s in r]), dev)
    base, rope = new(len(spans)), new(3, T)
    pkv.rope_spans(scu, spans, base)
    pkv.rope_positions(pos, seq, scu, spans, base, rope)
    qstride = (2 * Hq + 2 * Hkv) * D
    qkv = torch.randn(T, qstride, device=dev, generator=g).bfloat16()
    q = qkv[:, :2 * Hq * D].view(T, Hq, 2, D)
    k, v = qkv[:, 2 * Hq * D:].view(T, 2, Hkv, D).unbind(1)
    half = 32
    axes = i32([i % 3 for i in range(half)], dev)
    inv = (1e7 ** (-torch.arange(half, device=dev) / half)).float()
    w = 1.0 + 0.1 * torch.randn(D, device=dev, generator=g)
    qr, kr = torch.empty(T, Hq, D, device=dev, dtype=torch.bfloat16), torch.empty(T, Hkv, D, device=dev, dtype=torch.bfloat16)
    pkv.rope_rows(q[:, :, 0], k, rope, axes, inv, qr, kr, q_norm=w, k_norm=w)
    kc, vc = (torch.zeros(pool * bs, Hkv, D, device=dev, dtype=torch.bfloat16) for _ in range(2))
    vr = v.contiguous()
    pkv.append(kr, vr, Hkv * D * 2, slot, T, Hkv, D * 2, kc, vc, pool * bs)
    assert torch.equal(kc[slot.long()], kr)
    out, packed = torch.zeros_like(qr), torch.zeros_like(qr)
    pkv.attn_prefill(qr, kc, vc, qkv, qstride, Hq, Hkv, pos, cu, n, table, width, bs, out, 1 / 16, None, 1, T, pool)
    pkv.attn_packed(qr, kr, v, cu, packed, 1 / 16, gate=q[:, :, 1])
    prompts = torch.ones(T, dtype=torch.bool, device=dev)
    prompts[70] = False  # one token: the paged prompt kernel leaves it to decode
    near = 2.0 ** -4 * float(v.float().abs().max())
    assert ((out.float() - packed.float()).abs()[prompts] <= near).all()
    assert (out.float() - packed.float())[prompts].norm() <= 0.02 * packed.float()[prompts].norm()
    # the next step: one token each, its position behind the images
    pos1, slot1, seq1, cu1 = new(n), new(n), new(n), new(n + 1)
    pkv.plan_step(length, held, i32([1] * n, dev), table, bs, pool, pos1, slot1, seq1, cu1, limits, length, held, status,
                  free_list=free, free_count=count, free_count_out=count)
    assert pos1.tolist() == lens and not status.any()
    rope1 = new(3, n)
    pkv.rope_positions(pos1, seq1, scu, spans, base, rope1)
    assert rope1[:, 0].tolist() == [70 - 35 + 7] * 3 and rope1[:, 3].tolist() == [30, 30, 33]
    row = torch.randn(n, qstride, device=dev, generator=g).bfloat16()
    q1 = row[:, :2 * Hq * D].view(n, Hq, 2, D)
    k1, v1 = row[:, 2 * Hq * D:].view(n, 2, Hkv, D).unbind(1)
    q1r, k1r = torch.empty(n, Hq, D, device=dev, dtype=torch.bfloat16), torch.empty(n, Hkv, D, device=dev, dtype=torch.bfloat16)
    pkv.rope_rows(q1[:, :, 0], k1, rope1, axes, inv, q1r, k1r, q_norm=w, k_norm=w)
    ws = torch.empty(pkv.attn_decode_workspace(n, Hq), dtype=torch.uint8, device=dev)
    o1 = torch.zeros(n, Hq, D, device=dev, dtype=torch.bfloat16)
    pkv.append(k1r, v1.contiguous(), Hkv * D * 2, slot1, n, Hkv, D * 2, kc, vc, pool * bs)
    pkv.attn_decode(q1r, kc, vc, row, qstride, Hq, Hkv, pos1, seq1, table, width, bs, o1, 1 / 16, cu1, False, None, 1, n,
                    pool, ws)
    # the same rows as the last of packed prompts that hold everything
    at = np.concatenate([[0], np.cumsum(lens)])
    full = lambda a, b: torch.cat([torch.cat([a[at[s]:at[s + 1]], b[s:s + 1]]) for s in range(n)])
    fq, fk, fv, fg = full(qr, q1r), full(kr, k1r), full(v, v1), full(q[:, :, 1], q1[:, :, 1])
    fcu = i32(at + np.arange(n + 1), dev)
    fo = torch.zeros_like(fq)
    pkv.attn_packed(fq, fk, fv, fcu, fo, 1 / 16, gate=fg)
    last = fo[fcu[1:].long() - 1]
    assert ((o1.float() - last.float()).abs() <= near).all()
    assert (o1.float() - last.float()).norm() <= 0.02 * last.float().norm()


def test_a_captured_prompt_step(dev):
    """Plan, positions, rows and attention of a batch of prompts captured once, replayed for other lengths and values
    with eager calls between: every replay equal to the eager run of the same step."""
    n, T, Hq, Hkv, D, bs, pool, width = 5, 400, 8, 2, 128, 16, 80, 30
    g = torch.Generator(device=dev).manual_seed(9)
    new = lambda *k: torch.zeros(*k, dtype=torch.int32, device=dev)
    rows = lambda h: torch.zeros(T, h, D, device=dev, dtype=torch.bfloat16)
    scu, spans = i32([0, 1, 1, 3, 3, 3], dev), i32([[4, 1, 3, 5, 1], [0, 2, 2, 2, 3], [30, 1, 4, 6, 1]], dev)
    axes = i32([i % 3 for i in range(D // 2)], dev)
    inv = (1e6 ** (-torch.arange(D // 2, device=dev) / (D // 2))).float()
    ntok, free = new(n), i32(np.random.default_rng(2).permutation(pool), dev)
    count, zero = i32([pool], dev), new(n)
    q, k, v = rows(Hq), rows(Hkv), rows(Hkv)

    def buffers():
        return dict(table=new(n, width), pos=new(T), slot=new(T), seq=new(T), cu=new(n + 1), limits=new(n), len=new(n),
                    held=new(n), left=new(1), status=new(n), base=new(3), rope=new(3, T), q=rows(Hq), k=rows(Hkv),
                    out=rows(Hq))

    def step(b):
        pkv.plan_step(zero, zero, ntok, b["table"], bs, pool, b["pos"], b["slot"], b["seq"], b["cu"], b["limits"], b["len"],
                      b["held"], b["status"], free_list=free, free_count=count, free_count_out=b["left"])
        pkv.rope_spans(scu, spans, b["base"])
        pkv.rope_positions(b["pos"], b["seq"], scu, spans, b["base"], b["rope"])
        pkv.rope_rows(q, k, b["rope"], axes, inv, b["q"], b["k"])
        pkv.attn_packed(b["q"], b["k"], v, b["cu"], b["out"], D ** -0.5)

    one, two = buffers(), buffers()
    step(one)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        step(one)
    for lens in ([100, 0, 250, 1, 49], [1, 1, 1, 1, 1], [400, 0, 0, 0, 0], [-20, 30, 60, -100, 8], [0, 0, 0, 0, 0]):
        ntok.copy_(i32(lens, dev))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=dev, generator=g))
        for b in (one, two):
            for x in b.values():
                x.zero_()
        graph.replay()
        step(two)
        torch.cuda.synchronize()
        for name in one:
            assert torch.equal(one[name], two[name]), (lens, name)
        assert one["cu"].tolist() == np.concatenate([[0], np.cumsum(np.abs(lens))]).tolist()
        used = int(one["cu"][-1])
        assert (one["out"][used:] == 0).all() and (one["slot"][used:] == -1).all()
