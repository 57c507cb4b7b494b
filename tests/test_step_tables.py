"""Step tables built on the GPU from request lengths (cache.build_step) against a plain Python
walk over the requests, and the entry point's refusals."""
import ctypes as C
import random

import pytest
import torch


def walk(ctx, new, table, free, bs, n_slots, head=0):
    """Tables of a step request by request, token by token (plain integers)."""
    table = [row[:] for row in table]
    most = len(table[0]) if table else 0
    starts, lens, slots, positions, taken = [0], [], [], [], 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        blocks = lambda x: min(-(-x // bs), most)
        for e in range(blocks(c), blocks(c + n)):
            at = max(head, 0) + taken
            table[s][e] = free[at] if at < len(free) else -1
            taken += 1
        for pos in range(c, c + n):
            e = pos // bs
            block = table[s][e] if e < most else -1
            slots.append(block * bs + pos % bs if block >= 0 else -1)
            positions.append(pos)
        starts.append(starts[-1] + n)
        lens.append(c + n)
    pad = n_slots - len(slots)
    slots, positions = slots + [-1] * pad, positions + [0] * pad
    return starts, lens, slots[:n_slots], positions[:n_slots], taken, table


def check(dev, ctx, new, bs, max_blocks, n_free, *, pad=0, head=None, seed=0, strided=False):
    from knlp_b200 import cache
    rng = random.Random(seed)
    S = len(ctx)
    table = [[rng.randrange(10 ** 6) for _ in range(max_blocks)] for _ in range(S)]
    free = [rng.randrange(2 ** 20, 2 ** 27) for _ in range(n_free)]
    n_slots = sum(max(n, 0) for n in new) + pad
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).to(dev)
    wide = torch.full((S, max_blocks + (5 if strided else 0)), 77, dtype=torch.int32, device=dev)
    bt = wide[:, :max_blocks]
    bt.copy_(i32(table).view(S, max_blocks))
    t = cache.build_step(i32(ctx), i32(new), bt, i32(free), bs, n_slots,
                         free_head=None if head is None else i32([head]))
    starts, lens, slots, positions, taken, want = walk(ctx, new, table, free, bs, n_slots, head or 0)
    assert t.query_start_loc.tolist() == starts
    assert t.seq_lens.tolist() == lens
    assert t.blocks_taken.tolist() == [taken]
    assert t.slot_mapping.tolist() == slots
    assert t.positions.tolist() == positions
    assert bt.tolist() == want
    assert (wide[:, max_blocks:] == 77).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [1, 16, 48])
@pytest.mark.parametrize("seqs,q_hi", [(1, 1), (1, 5000), (37, 1), (33, 90), (1025, 3), (2600, 2)])
def test_against_the_walk(bs, seqs, q_hi, cuda_device):
    rng = random.Random(bs * 1000 + seqs)
    ctx = [rng.choice((0, 0, 1, bs, bs - 1, bs + 1, rng.randint(0, 400))) for _ in range(seqs)]
    new = [rng.randint(0 if seqs > 1 else q_hi, q_hi) for _ in range(seqs)]
    max_blocks = -(-(max(ctx) + q_hi) // bs)
    wanted = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(ctx, new))
    check(cuda_device, ctx, new, bs, max_blocks, wanted + 3, pad=rng.choice((0, 1, 255)), seed=seqs)


@pytest.mark.gpu
def test_edges(cuda_device):
    dev = cuda_device
    check(dev, [5, 0, 40], [0, 0, 0], 16, 4, 0)  # nothing new
    check(dev, [5, 0, 40], [0, 0, 0], 16, 4, 3, pad=7)
    check(dev, [0] * 40, [17] * 40, 16, 2, 30)  # the free list ends in the middle of the batch
    check(dev, [0] * 40, [17] * 40, 16, 2, 100, head=20)  # and with a front of its own
    check(dev, [0] * 4, [17] * 4, 16, 2, 6, head=-3)
    check(dev, [0] * 4, [17] * 4, 16, 2, 6, head=9)
    check(dev, [20, 3, 60], [30, 70, 1], 16, 3, 20)  # rows too short for their tokens
    check(dev, [-5, 3, -1], [4, -2, -7], 16, 3, 20)  # negative lengths count as 0
    check(dev, [9, 30, 2], [40, 3, 8], 16, 6, 20, strided=True)


@pytest.mark.gpu
def test_no_requests_and_corrupt_lengths(cuda_device):
    from knlp_b200 import cache
    dev = cuda_device
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32).to(dev)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    t = cache.build_step(none, none, torch.empty(0, 4, dtype=torch.int32, device=dev), none, 16, 5)
    assert t.query_start_loc.tolist() == [0] and t.blocks_taken.tolist() == [0]
    assert t.slot_mapping.tolist() == [-1] * 5 and t.positions.tolist() == [0] * 5
    # lengths near 2^31: useless tables, but nothing outside the rows is touched
    big = 2 ** 31 - 1
    wide = torch.full((6, 8), 55, dtype=torch.int32, device=dev)
    cache.build_step(i32(big, 0, big, 3, 0, big), i32(big, big, 1, big, big, 0), wide[:, 2:6],
                     i32(*range(40)), 16, 100)
    assert (wide[:, :2] == 55).all() and (wide[:, 6:] == 55).all()


@pytest.mark.gpu
def test_in_a_graph_with_new_lengths(cuda_device):
    """A captured step reads the lengths, the free list's front and the table at replay."""
    from knlp_b200 import cache
    dev = cuda_device
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).to(dev)
    ctx, new, head = i32([3, 40]), i32([2, 1]), i32([0])
    bt = torch.zeros(2, 8, dtype=torch.int32, device=dev)
    free = torch.arange(100, 140, dtype=torch.int32, device=dev)
    cache.build_step(ctx, new, bt, free, 16, 64, free_head=head)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t = cache.build_step(ctx, new, bt, free, 16, 64, free_head=head)
        head += t.blocks_taken
    table, at = [[0] * 8 for _ in range(2)], 0
    for c, n in (([0, 0], [20, 1]), ([20, 1], [1, 33]), ([21, 34], [12, 0])):
        ctx.copy_(i32(c)); new.copy_(i32(n)); bt.copy_(i32(table)); head.fill_(at)
        g.replay()
        starts, lens, slots, pos, taken, table = walk(c, n, table, free.tolist(), 16, 64, at)
        at += taken
        assert t.slot_mapping.tolist() == slots and t.seq_lens.tolist() == lens
        assert bt.tolist() == table and head.tolist() == [at]


def test_refusals_of_the_library():
    from knlp_b200 import _lib
    lib = _lib.load()
    buf = C.create_string_buffer(64)
    p = C.cast(buf, C.c_void_p)

    def call(**kw):
        a = dict(ctx=p, new=p, bt=p, stride=4, blocks=4, free=p, n_free=4, head=None, seqs=2,
                 bs=16, slots=8, starts=p, lens=p, map=p, pos=None, taken=p)
        a.update(kw)
        return lib.knlp_b200_build_step(*a.values(), None)

    for missing in ("ctx", "new", "bt", "free", "starts", "lens", "map", "taken"):
        assert call(**{missing: None}) == -1, missing
    for bad in (dict(seqs=-1), dict(slots=-1), dict(n_free=-1), dict(bs=0), dict(blocks=0)):
        assert call(**bad) == -2
    assert call(stride=3) == -5
    assert call(slots=1 << 30) == -9 and call(blocks=(1 << 20) + 1, stride=1 << 21) == -9


def test_cpu_tensors_are_refused():
    from knlp_b200 import cache
    v = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        cache.build_step(v, v, torch.zeros(2, 4, dtype=torch.int32), v, 16, 4)


@pytest.mark.gpu
def test_refusals_of_the_wrapper(cuda_device):
    from knlp_b200 import cache
    dev = cuda_device
    v = torch.ones(2, dtype=torch.int32, device=dev)
    bt = torch.zeros(2, 4, dtype=torch.int32, device=dev)
    for a in ((v.long(), v, bt, v), (v, v.long(), bt, v), (v, v, bt.long(), v), (v, v, bt, v.long())):
        with pytest.raises(TypeError):
            cache.build_step(*a, 16, 4)
    for a in ((v[:1], v, bt, v), (v, v[:1], bt, v), (v, v, bt[:1], v), (v, v, bt.t(), v),
              (v, v, bt[:, :0], v), (v[None], v, bt, v)):
        with pytest.raises(ValueError):
            cache.build_step(*a, 16, 4)
    with pytest.raises(ValueError):
        cache.build_step(v, v, bt, v, 0, 4)
    with pytest.raises(ValueError):
        cache.build_step(v, v, bt, v, 16, -1)
