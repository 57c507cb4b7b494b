"""Attention of several query tokens per sequence over the packed cache, against softmax in 64
bits over the dequantized values, with bounds derived from the roundings that the kernels make."""
import ctypes as C
import math
import random

import pytest
import torch

MODES = ("int4_asym", "int4_sym", "k8v4", "k8v4_sym", "k8v8", "kfpv4", "kfpv4_sym", "kfpv8")
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _codes(x, bits, asym):
    g = x.unflatten(-1, (-1, 32))
    if bits == 8:
        s = g.abs().amax(-1, keepdim=True) / 127 + 1e-9
        return torch.round(g / s).clamp(-128, 127).to(torch.int8).flatten(-2), s.squeeze(-1).half(), None
    if asym:
        lo = g.amin(-1, keepdim=True)
        s = (g.amax(-1, keepdim=True) - lo).clamp_min(1e-8) / 15
        q, z = torch.round((g - lo) / s).clamp(0, 15), lo.squeeze(-1).half()
    else:
        s = g.abs().amax(-1, keepdim=True) / 7 + 1e-9
        q, z = torch.round(g / s).clamp(-8, 7) + 8, None
    q = q.flatten(-2).to(torch.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), s.squeeze(-1).half(), z


def _values(codes, s, z):
    if s is None:
        return codes.double()
    if codes.dtype == torch.uint8:
        c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double() - (8 if z is None else 0)
    else:
        c = codes.double()
    c = c * s.double().repeat_interleave(32, -1)
    return c if z is None else c + z.double().repeat_interleave(32, -1)


class Batch:
    """A paged cache of random K / V in one mode, with ragged sequences on shuffled pages."""

    def __init__(self, dev, ctx, new, hq, hkv, d, mode, q="bf16", bs=16, seed=0, spare=3,
                 pad_rows=0, layout="natural"):
        g = torch.Generator().manual_seed(seed)
        lens = [c + n for c, n in zip(ctx, new)]
        pages = [-(-n // bs) for n in lens]
        nb = max(1, sum(pages)) + 2
        kd = DT[q]
        wide = torch.where(torch.rand(hkv, d, generator=g) < 0.02, 8.0, 1.0)
        k = torch.randn(nb, bs, hkv, d, generator=g) * wide * 0.6
        v = torch.randn(nb, bs, hkv, d, generator=g) + torch.randn(hkv, d, generator=g)
        asym = not mode.endswith("sym") or mode == "int4_asym"
        if mode.startswith("kfp"):
            self.k, self.ks, self.kz = k.to(kd), None, None
        else:
            self.k, self.ks, self.kz = _codes(k, 8 if mode.startswith("k8") else 4, asym)
        v8 = mode.endswith("v8")
        self.v, self.vs, self.vz = _codes(v, 8 if v8 else 4, asym)
        self.mode, self.asym = mode, asym and not v8 or mode == "int4_asym"
        self.hq, self.hkv, self.d, self.bs = hq, hkv, d, bs
        perm = torch.randperm(nb, generator=g).tolist()
        cols = max(1, max(pages, default=1)) + spare
        table = torch.full((len(ctx), cols), -7, dtype=torch.int32)  # entries nobody may follow
        at = 0
        for i, p in enumerate(pages):
            table[i, :p] = torch.tensor(perm[at:at + p], dtype=torch.int32)
            at += p
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        query = torch.randn(starts[-1] + pad_rows, hq, d, generator=g).to(DT[q])
        self.T = starts[-1]

        def lay(t):
            if t is None:
                return None
            t = t.to(dev)
            if layout == "natural":
                return t
            if layout == "head_major":  # [blocks, heads, block, ..] underneath
                return t.transpose(1, 2).contiguous().transpose(1, 2)
            w = torch.zeros(t.shape[0], t.shape[1], t.shape[2] + 1, t.shape[3] + (
                8 if layout == "padded" else 1), dtype=t.dtype, device=dev)
            w = w[:, :, 1:, :t.shape[3]]  # rows wider than they need; "odd": unaligned ones
            w.copy_(t)
            return w
        for name in ("k", "ks", "kz", "v", "vs", "vz"):
            setattr(self, name, lay(getattr(self, name)))
        self.table, self.query = table.to(dev), query.to(dev)
        self.lens = torch.tensor(lens, dtype=torch.int32).to(dev)
        self.starts = torch.tensor(starts, dtype=torch.int32).to(dev)

    def run(self, **kw):
        from knlp_b200 import ops
        m = self.mode
        rest = (self.table, self.lens, self.starts, self.hkv, self.d)
        vz = dict(v_zeros=self.vz, asymmetric=self.asym)
        if m.startswith("int4"):
            return ops.fused_int4_extend(self.query, self.k, self.v, self.ks, self.vs, *rest,
                                         k_zeros=self.kz, **vz, **kw)
        if m == "k8v8":
            return ops.kint8_vint8_extend(self.query, self.k, self.v, self.ks, self.vs, *rest, **kw)
        if m == "kfpv8":
            return ops.kfp16_vint8_extend(self.query, self.k, self.v, self.vs, *rest, **kw)
        if m.startswith("k8"):
            return ops.kint8_vint4_extend(self.query, self.k, self.v, self.ks, self.vs, *rest, **vz, **kw)
        return ops.kfp16_vint4_extend(self.query, self.k, self.v, self.vs, *rest, **vz, **kw)

    def reference(self, causal=True, scale=None, without=()):
        """(o, lse, bound of o, bound of lse) in 64 bits, rows [T, hq], `without` tokens at some
        positions.

        The bound: K and V are rounded to fp16 after dequantization, a bf16 Q below 2^-14 and P
        to fp16 (each within 2^-11 of its value or 2^-25), products are summed in fp32,
        exponentials are good to 2^-20.  A score is then off by at most
        e = scale sum (|q k| (2^-11 + d 2^-24) + |k| 2^-25 + |q| 2^-25),
        which changes every normalized weight by at most a factor exp(2e); so o is within
        (exp(2e) - 1 + 2 * 2^-11 + 2^-18) sum p |v| + n 2^-25 max|v|, and lse within e + 2^-18."""
        dev = self.query.device
        scale = self.d ** -0.5 if scale is None else scale
        rows = self.query.shape[0]
        o = torch.zeros(rows, self.hq, self.d, dtype=torch.float64, device=dev)
        lse = torch.full((rows, self.hq), -math.inf, dtype=torch.float64, device=dev)
        bo, bl = torch.zeros_like(o), torch.zeros_like(lse)
        kv, vv = _values(self.k, self.ks, self.kz), _values(self.v, self.vs, self.vz)
        rep = self.hq // self.hkv
        starts, lens = self.starts.tolist(), self.lens.tolist()
        for s, n in enumerate(lens):
            a, b = starts[s], starts[s + 1]
            n = min(n, self.table.shape[1] * self.bs)
            if b <= a or n <= 0:
                continue
            blocks = self.table[s, :-(-n // self.bs)].long()
            k = kv[blocks].flatten(0, 1)[:n].repeat_interleave(rep, 1)
            v = vv[blocks].flatten(0, 1)[:n].repeat_interleave(rep, 1)
            q = self.query[a:b].double()
            w = torch.einsum("qhd,khd->hqk", q, k) * scale
            e = torch.einsum("qhd,khd->hqk", q.abs(), k.abs()) * (2.0 ** -11 + self.d * 2.0 ** -24)
            e = scale * (e + 2.0 ** -25 * (k.abs().sum(-1).t()[:, None] + q.abs().sum(-1).t()[..., None]))
            if causal:
                last = lens[s] - (b - a) + torch.arange(b - a, device=dev)
                off = torch.arange(n, device=dev)[None] > last[:, None]
                w, e = w.masked_fill(off, -math.inf), e.masked_fill(off, 0)
            w[..., list(without)], e[..., list(without)] = -math.inf, 0
            ls = torch.logsumexp(w, -1)
            p = torch.exp(w - torch.where(ls.isinf(), 0, ls)[..., None])
            worst = e.amax(-1)
            o[a:b] = torch.einsum("hqk,khd->qhd", p, v)
            lse[a:b] = ls.t()
            bo[a:b] = (torch.expm1(2 * worst) + 2 * 2.0 ** -11 + 2.0 ** -18).t()[..., None] * (
                torch.einsum("hqk,khd->qhd", p, v.abs())) + n * 2.0 ** -25 * (1 + v.abs().amax())
            bl[a:b] = worst.t() + 2.0 ** -18 * (1 + torch.where(ls.isinf(), 0, ls).abs().t())
        return o, lse, bo, bl

    def check(self, causal=True, scale=None, **kw):
        o, lse, bo, bl = self.reference(causal, scale)
        r, l = self.run(causal=causal, softmax_scale=scale, return_lse=True, **kw)
        T = self.T
        half = torch.finfo(r.dtype).eps / 2  # rounding of the result
        err = (r[:T].double() - o[:T]).abs()
        bad = err > bo[:T] + half * (o[:T].abs() + bo[:T])
        assert not bad.any(), f"{int(bad.sum())} values off, worst {float((err / bo[:T].clamp_min(1e-30)).max()):.3g} bounds"
        fin = lse[:T].isfinite()
        assert torch.equal(l[:T].isfinite(), fin) and (l[:T][~fin] == -math.inf).all()
        assert ((l[:T].double() - lse[:T]).abs()[fin] <= bl[:T][fin]).all()
        assert (r[:T][~fin] == 0).all()
        from knlp_b200 import ops
        assert ops.device_status() == 0  # no wait inside a kernel ran out
        return r


GENERIC = [False, True]


@pytest.mark.gpu
@pytest.mark.parametrize("generic", GENERIC)
@pytest.mark.parametrize("q", ["bf16", "f16"])
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (6, 6, 64)])
def test_modes(mode, q, hq, hkv, d, generic, cuda_device):
    b = Batch(cuda_device, [0, 5, 130, 300, 17], [1, 40, 3, 150, 0], hq, hkv, d, mode, q, seed=1)
    b.check(force_generic=generic)
    b.check(force_generic=generic, out_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("generic", GENERIC)
@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 64), (5, 1, 128), (12, 4, 64), (16, 2, 128), (40, 1, 64),
                                      (130, 1, 64), (300, 1, 128), (7, 7, 128), (4, 2, 32), (6, 2, 256)])
def test_head_layouts(hq, hkv, d, generic, cuda_device):
    Batch(cuda_device, [100, 0, 3], [9, 70, 1], hq, hkv, d, "int4_asym", seed=hq).check(
        force_generic=generic, out_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_every_length_around_the_tiles(d, cuda_device):
    """One new token, a few, and a whole prompt, at cached lengths around 0 and the tile ends."""
    edges = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 385]
    Batch(cuda_device, [n - 1 for n in edges], [1] * len(edges), 4, 1, d, "int4_asym", seed=5).check(
        out_dtype=torch.float32)
    Batch(cuda_device, [max(n - 7, 0) for n in edges], [min(n, 7) for n in edges], 8, 2, d, "k8v8",
          "f16", seed=6).check(out_dtype=torch.float32)
    Batch(cuda_device, [0] * len(edges), edges, 4, 2, d, "int4_sym", seed=7).check(
        out_dtype=torch.float32)
    Batch(cuda_device, [3] * len(edges), edges, 3, 1, d, "kfpv4", seed=8).check(
        out_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("ctx,new", [([5000], [1]), ([7001], [5]), ([3000], [700]), ([0], [1500]),
                                     ([9000, 10, 4000], [4, 4, 4]), ([6000] * 5, [1, 2, 33, 64, 65])])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (8, 8)])
def test_long_contexts_split_over_blocks(ctx, new, hq, hkv, cuda_device):
    Batch(cuda_device, ctx, new, hq, hkv, 128, "int4_asym", seed=11).check(out_dtype=torch.float32)


@pytest.mark.gpu
def test_ragged_batches(cuda_device):
    rng = random.Random(2)
    for seed in range(4):
        S = rng.choice((3, 20, 70))
        ctx = [rng.choice((0, 1, rng.randint(0, 900))) for _ in range(S)]
        new = [rng.choice((0, 1, 1, 2, rng.randint(1, 200))) for _ in range(S)]
        Batch(cuda_device, ctx, new, 8, 2, rng.choice((64, 128)), rng.choice(MODES), seed=seed).check()


@pytest.mark.gpu
def test_many_sequences_and_many_tiles(cuda_device):
    """More sequences and more row tiles than the planning keeps in shared memory."""
    rng = random.Random(5)
    S = 1300
    Batch(cuda_device, [rng.randint(0, 60) for _ in range(S)], [rng.choice((0, 1, 1, 1, 9)) for _ in range(S)],
          8, 2, 64, "int4_asym", seed=31).check()
    Batch(cuda_device, [rng.randint(0, 90) for _ in range(30)], [150] * 30, 128, 1, 64, "k8v8", seed=32).check()


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(8, 1), (4, 4), (32, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_row_counts_around_the_kernels_border(d, hq, hkv, cuda_device):
    """Rows per kv head (new tokens x q heads of a group) around 8, 16, 24, 32, 128 and 256, where the
    groups of the few-row kernel, the kernels and the tiles change."""
    rep = hq // hkv
    new = sorted({max(1, n // rep + k) for n in (8, 16, 24, 32, 128, 256, 288) for k in (-1, 0, 1)})
    rng = random.Random(d)
    Batch(cuda_device, [rng.choice((0, 5, 127, 300, 900)) for _ in new], new, hq, hkv, d, "int4_asym",
          seed=33).check(out_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("hints", [dict(max_query_len=1), dict(max_seq_len=1), dict(max_query_len=1, max_seq_len=1),
                                   dict(max_query_len=0, max_seq_len=0), dict(max_query_len=9, max_seq_len=10 ** 6),
                                   dict(max_query_len=10 ** 6, max_seq_len=300)])
def test_the_hosts_bounds_do_not_change_the_result(hints, cuda_device):
    """Bounds that are right, too small or too large."""
    Batch(cuda_device, [3000, 0, 700, 5, 130], [9, 400, 1, 0, 33], 8, 2, 128, "int4_asym", seed=34).check(
        out_dtype=torch.float32, **hints)
    Batch(cuda_device, [100, 300, 20], [2, 1, 4], 8, 2, 64, "k8v8", seed=35).check(**hints)


@pytest.mark.gpu
@pytest.mark.parametrize("generic", GENERIC)
def test_full_and_scale(generic, cuda_device):
    """Every query token over all cached tokens; other scales than head_dim^-1/2."""
    b = Batch(cuda_device, [300, 40, 0], [20, 1, 60], 8, 2, 128, "int4_asym", seed=3)
    b.check(causal=False, force_generic=generic, out_dtype=torch.float32)
    b.check(scale=0.02, force_generic=generic, out_dtype=torch.float32)
    b.check(causal=False, scale=0.3, force_generic=generic, out_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("generic", GENERIC)
def test_rows_that_attend_to_nothing(generic, cuda_device):
    """Fewer cached tokens than new ones (their first rows see nothing), empty sequences, lengths
    below 0 and beyond the table's row."""
    dev = cuda_device
    b = Batch(dev, [40, 0, 200, 30, 64], [10, 30, 0, 100, 3], 8, 2, 128, "int4_asym", seed=4, spare=0)
    b.lens = torch.tensor([50, 12, 200, 0, 40000], dtype=torch.int32, device=dev)
    # the last sequence's length is cut at its row of the table, the positions are not moved
    b.table[4] = b.table[2]
    b.check(force_generic=generic, out_dtype=torch.float32)
    b.lens[3] = -5
    b.check(force_generic=generic, out_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("generic", GENERIC)
@pytest.mark.parametrize("layout", ["natural", "head_major", "padded", "odd"])
@pytest.mark.parametrize("mode", ["int4_asym", "k8v4", "kfpv8"])
def test_layouts(mode, layout, generic, cuda_device):
    b = Batch(cuda_device, [70, 0, 300], [5, 90, 1], 8, 2, 128, mode, seed=9, layout=layout)
    b.check(force_generic=generic)


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [1, 8, 16, 24, 64, 128, 256])
def test_block_sizes(bs, cuda_device):
    Batch(cuda_device, [0, 100, 257], [130, 3, 1], 8, 2, 64, "int4_asym", bs=bs, seed=bs).check()


@pytest.mark.gpu
@pytest.mark.parametrize("generic", GENERIC)
def test_query_strides_and_rows_behind_the_last_sequence(generic, cuda_device):
    b = Batch(cuda_device, [20, 150], [50, 4], 8, 2, 128, "int4_asym", seed=12, pad_rows=11)
    wide = torch.zeros(b.query.shape[0], 3, 8, 130, dtype=b.query.dtype, device=cuda_device)
    wide[:, 1, :, 2:] = b.query
    out = torch.full((65, 8, 128), 7.5, dtype=torch.float32, device=cuda_device)
    b.check(force_generic=generic, out=out)
    assert (out[54:] == 7.5).all()
    for view in (wide[:, 1, :, 2:], torch.flip(b.query, [1]).flip(1)[:, :], b.query.transpose(0, 1).contiguous().transpose(0, 1)):
        b.query = view
        b.check(force_generic=generic)


@pytest.mark.gpu
@pytest.mark.parametrize("generic", GENERIC)
def test_bad_table_entries_do_not_fault(generic, cuda_device):
    """Entries outside the cache are clamped to it (as the decode does); whatever lies in a
    block behind a sequence's end (NaN scales here) changes nothing."""
    b = Batch(cuda_device, [90, 30], [10, 7], 8, 2, 128, "int4_asym", seed=13)
    nan = torch.tensor(math.nan, dtype=torch.float16, device=cuda_device)
    used = torch.zeros(b.k.shape[0] * b.bs, dtype=torch.bool, device=cuda_device)
    for s, n in enumerate(b.lens.tolist()):
        t = torch.arange(n, device=cuda_device)
        used[b.table[s, t // b.bs].long() * b.bs + t % b.bs] = True
    for plane in (b.ks, b.kz, b.vs, b.vz):
        plane.view(-1, *plane.shape[2:])[~used] = nan
    b.check(force_generic=generic)
    b.table[0, 2], b.table[1, 0] = 1 << 30, -(1 << 30)
    b.run(force_generic=generic)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("generic", GENERIC)
@pytest.mark.parametrize("mode,many", [("int4_asym", False), ("k8v8", False), ("int4_sym", False),
                                       ("int4_asym", True)])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(mode, many, generic, cuda_device):
    """An overflowed scale or zero-point of V belongs to the rows that attend to its token: rows
    before it (the mask leaves 0 x NaN there) are as if it were not."""
    b = Batch(cuda_device, [40, 300], [200, 5], 8, 2, 128, mode, seed=17)
    o, _, bo, _ = b.reference()
    T, at = b.T, 40 + 90  # the token at position 130 of the first sequence, its kv head 1, group 2
    tokens = range(at, at + 40) if many else (at,)
    for t in tokens:
        blk, off = int(b.table[0, t // 16]), t % 16
        b.vs[blk, off, 1, 2] = math.inf
        if b.vz is not None:
            b.vz[blk, off, 1, 2] = -math.inf
    if mode == "int4_sym":
        b.vs[blk, off, 1, 2] = math.nan  # inf x code would be inf or NaN by the code
    elif mode == "k8v8":
        b.vs[blk, off, 1, 2] = math.nan
    r = b.run(force_generic=generic, out_dtype=torch.float32).double()
    see = torch.zeros(T, 8, 128, dtype=torch.bool, device=cuda_device)
    see[90:200, 4:, 64:96] = True
    fine = (r - o).abs() <= bo + 2.0 ** -23 * o.abs()
    assert torch.isnan(r[see]).all()
    assert fine[~see].all()


@pytest.mark.gpu
@pytest.mark.parametrize("generic", GENERIC)
@pytest.mark.parametrize("ctx,new,first", [(200, 3, 4), (200, 150, 4), (5000, 3, 200), (700, 3, 129),
                                           (300, 150, 129)])
def test_scores_of_minus_infinity_weigh_nothing(ctx, new, first, generic, cuda_device):
    """Keys that are -inf in one element, under queries that are positive there: as if their
    tokens were masked, wherever they lie (the first tokens, whole tiles, a run within one)."""
    b = Batch(cuda_device, [ctx], [new], 4, 2, 64, "kfpv8", "f16", seed=18)
    b.query[..., 7] = b.query[..., 7].abs() + 0.125
    hit = list(range(first)) + [first + 1, 64] + list(range(130, 150))
    o, lse, bo, bl = b.reference(without=hit)
    for t in hit:
        b.k[int(b.table[0, t // 16]), t % 16, :, 7] = -math.inf
    r, l = b.run(force_generic=generic, return_lse=True, out_dtype=torch.float32)
    assert ((r.double() - o).abs() <= bo + 2.0 ** -24 * (o.abs() + bo)).all()
    assert ((l.double() - lse).abs() <= bl).all()


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda_device):
    """A cache whose code planes pass 2^32 bytes, the sequence on its first and last blocks."""
    from knlp_b200 import ops
    dev, d, hkv, bs = cuda_device, 128, 8, 16
    nb = (1 << 32) // (bs * hkv * d // 2) + 64
    b = Batch(dev, [100], [20], 16, hkv, d, "int4_asym", seed=14)
    n = 8
    pick = [0, nb - 1, 1, nb - 2, nb // 2, nb - 40, 7, nb - 3]
    old = b.table[0, :n].long()
    big = {}
    for name in ("k", "ks", "kz", "v", "vs", "vz"):
        t = getattr(b, name)
        w = torch.empty((nb,) + t.shape[1:], dtype=t.dtype, device=dev)
        w[torch.tensor(pick, device=dev)] = t[old]
        big[name] = w
    o, _, bo, _ = b.reference()
    table = torch.tensor([pick], dtype=torch.int32, device=dev)
    r = ops.fused_int4_extend(b.query, big["k"], big["v"], big["ks"], big["vs"], table, b.lens,
                              b.starts, hkv, d, k_zeros=big["kz"], v_zeros=big["vz"],
                              asymmetric=True, out_dtype=torch.float32)
    assert ((r.double() - o).abs() <= bo + 2.0 ** -23 * o.abs()).all()


@pytest.mark.gpu
def test_large_scores_and_values(cuda_device):
    """Scores of several hundred (one key takes all the weight), values near fp16's largest."""
    b = Batch(cuda_device, [500], [70], 8, 2, 128, "k8v8", "f16", seed=15)
    b.query *= 30
    b.check(out_dtype=torch.float32)
    b = Batch(cuda_device, [500], [70], 8, 2, 128, "k8v8", "bf16", seed=16)
    b.vs.fill_(500.0)  # 127 x 500 = 63500
    b.check(out_dtype=torch.float32)


@pytest.mark.gpu
def test_streams_and_graphs(cuda_device):
    """The same call eagerly, on another stream at the same time, and captured: each has its own
    workspace, and a replay reads lengths and tables anew."""
    dev = cuda_device
    a = Batch(dev, [4000, 700], [6, 120], 8, 2, 128, "int4_asym", seed=20)
    b = Batch(dev, [2500], [300], 8, 2, 128, "int4_asym", seed=21)
    ra, rb = a.run(), b.run()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            got.append((a.run(), ra))
        with torch.cuda.stream(s2):
            got.append((b.run(), rb))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, y)
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        ca = a.run()
    with torch.cuda.graph(gb):
        cb = b.run()
    for _ in range(3):
        with torch.cuda.stream(s1):
            ga.replay()
        with torch.cuda.stream(s2):
            gb.replay()
    torch.cuda.synchronize()
    assert torch.equal(ca, ra) and torch.equal(cb, rb)
    a.lens -= 37  # shorter contexts in the same buffers
    ga.replay()
    torch.cuda.synchronize()
    assert torch.equal(ca, a.run())
    o, _, bo, _ = a.reference()
    assert ((ca.double() - o).abs() <= bo + torch.finfo(ca.dtype).eps / 2 * (o.abs() + bo)).all()


@pytest.mark.gpu
def test_threads_that_share_a_stream(cuda_device):
    """Calls of several host threads on one stream share its workspace; each call's launches stay
    together."""
    from concurrent.futures import ThreadPoolExecutor
    batches = [Batch(cuda_device, [3000 + 500 * i, 40], [5 + i, 90], 8, 2, 128, "int4_asym", seed=25 + i)
               for i in range(4)]
    want = [b.run() for b in batches]
    torch.cuda.synchronize()

    def calls(b):
        return [b.run() for _ in range(40)]
    with ThreadPoolExecutor(len(batches)) as pool:
        got = list(pool.map(calls, batches))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


@pytest.mark.gpu
def test_step_of_a_batch_through_the_cache(cuda_device):
    """The pieces as a server uses them: tables from lengths, write, attend, over several steps
    of prefill chunks, drafted tokens and single tokens; compared with the oracle's attention
    over everything written so far."""
    from knlp_b200 import cache, scoring
    dev, hq, hkv, d, bs = cuda_device, 8, 2, 128, 16
    g = torch.Generator().manual_seed(30)
    c = cache.PackedKVCache(hkv, d, "int8", "int4", asymmetric=True)
    c.ensure(200, bs, dev)
    builder = cache.AttentionMetadataBuilder(bs, hkv, d, dev)
    S, V = 3, 977
    table = torch.zeros(S, 40, dtype=torch.int32, device=dev)
    free = torch.randperm(200, generator=g).to(torch.int32).to(dev)
    head = torch.zeros(1, dtype=torch.int32, device=dev)
    w = (torch.randn(hq * d, V, generator=g) / 30).to(dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    ctx = [0, 0, 0]
    for new in ([130, 5, 64], [1, 1, 1], [1, 60, 4], [3, 0, 1], [1, 1, 1]):
        T = sum(new)
        q = torch.randn(T, hq, d, generator=g).to(torch.bfloat16).to(dev)
        k = torch.randn(T, hkv, d, generator=g).to(torch.bfloat16).to(dev)
        v = torch.randn(T, hkv, d, generator=g).to(torch.bfloat16).to(dev)
        meta, t = builder.build_from_lengths(
            i32(ctx), i32(new), table, free, num_tokens=T, max_query_len=max(new),
            max_seq_len=max(a + b for a, b in zip(ctx, new)), free_head=head)
        head += t.blocks_taken
        out = c.forward(q, k, v, meta, out_dtype=torch.float32)
        ctx = [a + b for a, b in zip(ctx, new)]
        assert t.seq_lens.tolist() == ctx
        b = Batch.__new__(Batch)
        b.k, b.ks, b.kz, b.v, b.vs, b.vz = (c.key_cache, c.k_scales, None, c.value_cache,
                                            c.v_scales, c.v_zeros)
        b.hq, b.hkv, b.d, b.bs, b.table, b.query = hq, hkv, d, bs, table, q
        b.lens, b.starts = t.seq_lens, t.query_start_loc
        o, _, bo, _ = b.reference()
        # single-token steps run the decode kernel, held to its own bar (2e-3 + 1e-3 |o|)
        slack = 2e-3 + 1e-3 * o.abs() if set(new) == {1} else 2.0 ** -23 * o.abs()
        assert ((out.double() - o).abs() <= bo + slack).all()
        # the scores of a sampled token for every row
        logits = out.view(T, hq * d) @ w
        ids = torch.randint(0, V, (T,), generator=g).to(dev)
        s = scoring.token_logprobs(logits, ids, top_k=4)
        want = torch.log_softmax(logits.double(), -1)
        assert (s.logprob.double() - want.gather(1, ids[:, None])[:, 0]).abs().max() < 1e-5
        assert torch.equal(s.top_logprobs[:, 0], s.top_logprobs.amax(-1))


def test_refusals_of_the_library():
    from knlp_b200 import _lib
    lib = _lib.load()
    buf = C.create_string_buffer(256)
    p = C.cast(buf, C.c_void_p).value
    st = (C.c_int64 * 2)(512, 128)

    def plane(mode):
        pl = _lib.KvPlane()
        pl.codes = pl.scales = pl.zeros = p
        pl.mode = mode
        return pl

    def call(**kw):
        a = dict(q=p, dt=2, st=st, k=C.byref(plane(2)), v=C.byref(plane(2)), bt=p, stride=4, blocks=4,
                 lens=p, starts=p, nb=9, S=0, T=0, hq=4, hkv=2, d=128, bs=16, mq=1, ms=64, scale=0.1,
                 ws=p, n=1 << 40, out=p, odt=2, row=128, lse=None, flags=0)
        a.update(kw)
        return lib.knlp_b200_extend_attention(*a.values(), None)

    assert call() == 0  # nothing to do
    for missing in ("q", "st", "k", "v", "bt", "lens", "starts", "ws", "out"):
        assert call(**{missing: None}) == -1, missing
    assert call(dt=0) == -3 and call(dt=9) == -3 and call(odt=5) == -3
    for bad in (dict(S=-1), dict(T=-1), dict(hq=5), dict(hkv=0), dict(d=96), dict(bs=0), dict(blocks=0),
                dict(nb=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(mq=-1), dict(ms=-1)):
        assert call(**bad) == -2, bad
    assert call(flags=64) == -4
    assert call(n=0) == -6
    assert call(row=127) == -5
    assert call(k=C.byref(plane(9))) == -4 and call(v=C.byref(plane(4))) == -4
    assert call(k=C.byref(plane(4))) == -4 and call(k=C.byref(plane(5)), dt=1) == -4
    none = plane(2)
    none.zeros = None
    assert call(k=C.byref(none)) == -1
    n = C.c_int64(0)
    assert lib.knlp_b200_extend_workspace(1, 1, 4, 2, 128, None) == -1
    assert lib.knlp_b200_extend_workspace(1, 1, 4, 3, 128, C.byref(n)) == -2
    assert lib.knlp_b200_extend_workspace(4, 100, 4, 2, 128, C.byref(n)) == 0 and n.value > 0


def test_cpu_tensors_are_refused():
    b = Batch("cpu", [3], [2], 2, 1, 64, "int4_asym")
    with pytest.raises(RuntimeError):
        b.run()


@pytest.mark.gpu
def test_refusals_of_the_wrapper(cuda_device):
    from knlp_b200 import ops
    b = Batch(cuda_device, [30, 9], [4, 5], 8, 2, 128, "int4_asym")
    good = dict(vars(b))

    def refuses(exc, **change):
        for key, val in change.items():
            setattr(b, key, val)
        with pytest.raises(exc):
            b.run()
        for key in change:
            setattr(b, key, good[key])

    refuses(TypeError, query=b.query.float())
    refuses(TypeError, lens=b.lens.long())
    refuses(TypeError, table=b.table.long())
    refuses(TypeError, starts=b.starts.long())
    refuses(TypeError, ks=b.ks.float())
    refuses(ValueError, starts=b.starts[:2])
    refuses(ValueError, table=b.table[:1])
    refuses(ValueError, query=b.query[0])
    refuses(ValueError, query=b.query[:, :7])
    refuses(ValueError, hkv=3)
    refuses(ValueError, k=b.k[..., :32])
    refuses(ValueError, vs=b.vs[..., :2])
    refuses(ValueError, v=b.v[:-1])
    refuses(RuntimeError, lens=b.lens.cpu())
    with pytest.raises(ValueError):
        b.run(out=torch.empty(9, 8, 64, device=cuda_device))
    with pytest.raises(RuntimeError):  # status of the library: the scale must be positive
        b.run(softmax_scale=-1.0)
    f = Batch(cuda_device, [30, 9], [4, 5], 8, 2, 128, "kfpv4", "f16")
    f.query = f.query.to(torch.bfloat16)
    with pytest.raises(TypeError):
        f.run()
