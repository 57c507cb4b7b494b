"""What a serving step over the packed KV cache does besides its single-token decode, as cases
that can be timed and compared:

  step    the step's tables from the requests' lengths: cache blocks taken from the free list,
          block-table entries, slot of every new token, positions, query offsets, lengths
  extend  attention of SEVERAL query tokens per sequence (chunked prefill, verification of
          drafted tokens, mixed batches) over a cache held in 4 bits (or 8, or with K as it is)
  score   log probability, entropy, rank and top alternatives of given tokens from logits

``run`` computes an operator in plain torch operations, or with ``own`` by the calls that a
user of knlp_b200 makes.
"""

import math
import random

import torch

own = False

PAGE = 16  # cache block size of the workloads of this repository
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a batch of 32 (the batch of the headline workload): a token each
        dict(name="step decode 32", op="step", seqs=32, max_blocks=2048, q_lo=1, q_hi=1,
             long_every=0, q_long=0, ctx_lo=1, ctx_hi=32000, lens=1),
        # a continuous batch: decodes with every 16th request prefilling a chunk
        dict(name="step mixed 256", op="step", seqs=256, max_blocks=2048, q_lo=1, q_hi=4,
             long_every=16, q_long=512, ctx_lo=0, ctx_hi=30000, lens=2),
        # admission of a large batch of whole prompts, 1.0 Mi new tokens
        dict(name="step prefill 1024", op="step", seqs=1024, max_blocks=256, q_lo=1, q_hi=2047,
             long_every=0, q_long=0, ctx_lo=0, ctx_hi=1900, lens=3),
        # one short sequence of the 12-head shape, a single new token: latency only
        dict(name="extend 12h single", op="extend", seqs=1, hq=12, hkv=12, d=64, mode="int4_sym",
             q="f16", q_lo=1, q_hi=1, long_every=0, q_long=0, ctx_lo=1000, ctx_hi=1000, lens=4),
        # verification of drafted tokens: up to 8 new tokens on long ragged contexts
        dict(name="extend verify 16", op="extend", seqs=16, hq=32, hkv=8, d=128, mode="int4_asym",
             q="bf16", q_lo=3, q_hi=8, long_every=0, q_long=0, ctx_lo=8000, ctx_hi=32000, lens=5),
        # mixed batch with the 8-bit-K cache: single tokens beside prefill chunks
        dict(name="extend mixed 32", op="extend", seqs=32, hq=32, hkv=8, d=128, mode="k8v4",
             q="bf16", q_lo=1, q_hi=1, long_every=8, q_long=500, ctx_lo=500, ctx_hi=4000, lens=6),
        # whole prompts of the 64-head shape, odd lengths, nothing cached before
        dict(name="extend prompts 4", op="extend", seqs=4, hq=64, hkv=8, d=128, mode="int4_asym",
             q="bf16", q_lo=1500, q_hi=3900, long_every=0, q_long=0, ctx_lo=0, ctx_hi=0, lens=7),
        # a prefill chunk deep in a long prompt
        dict(name="extend chunk 4096 at 28k", op="extend", seqs=1, hq=32, hkv=8, d=128,
             mode="int4_asym", q="bf16", q_lo=4096, q_hi=4096, long_every=0, q_long=0,
             ctx_lo=28000, ctx_hi=28000, lens=8),
        # head dimension 64 without grouped heads, both planes in 8 bits
        dict(name="extend 12h prompts k8v8", op="extend", seqs=8, hq=12, hkv=12, d=64, mode="k8v8",
             q="f16", q_lo=700, q_hi=2000, long_every=0, q_long=0, ctx_lo=0, ctx_hi=900, lens=9),
        # the token sampled for each of four sequences, with its alternatives
        dict(name="score 4", op="score", rows=4, vocab=50257, logits="f32", top=5, masked=0.0),
        # a decode batch whose grammar allows a tenth of the vocabulary
        dict(name="score 128 masked", op="score", rows=128, vocab=128256, logits="bf16", top=20,
             masked=0.9),
        # every token of a long prompt, as perplexity evaluation reads them
        dict(name="score 2047 prompt", op="score", rows=2047, vocab=50257, logits="bf16", top=8,
             masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("step", "extend", "extend", "score"))
    if op == "step":
        c = dict(op=op, seqs=_log_int(rng, 1, 1024), max_blocks=2048, q_lo=1, long_every=0,
                 q_long=0, ctx_lo=0, ctx_hi=_log_int(rng, 1, 30000), lens=rng.randrange(1 << 30))
        c["q_hi"] = _log_int(rng, 1, max(1, min(2000, 1000000 // c["seqs"])))
        return c
    if op == "score":
        vocab = _log_int(rng, 1000, 131072)
        rows = _log_int(rng, 1, max(1, min(4096, 100_000_000 // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, logits=rng.choice(("f32", "bf16", "f16")),
                    top=rng.choice((0, 1, 5, 8, 20, 32)), masked=rng.choice((0.0, 0.0, 0.9)))
    hq, hkv, d = rng.choice(((12, 12, 64), (32, 8, 128), (64, 8, 128), (32, 32, 128), (24, 8, 64)))
    mode = rng.choice(("int4_asym", "int4_asym", "int4_sym", "k8v4", "k8v8", "kfpv4", "kfpv8"))
    c = dict(op=op, hq=hq, hkv=hkv, d=d, mode=mode, q=rng.choice(("bf16", "f16")), long_every=0,
             q_long=0, lens=rng.randrange(1 << 30))
    kind = rng.choice(("single", "verify", "chunk", "mixed"))
    c["seqs"] = _log_int(rng, 1, 8 if kind == "chunk" else 32)
    c["q_lo"], c["q_hi"] = {"single": (1, 1), "verify": (2, 8), "mixed": (1, 4),
                            "chunk": (16, _log_int(rng, 32, 2000))}[kind]
    if kind == "mixed":
        c["long_every"], c["q_long"] = rng.choice((2, 5, 9)), _log_int(rng, 16, 600)
    # the plain form holds every score (seqs x heads x longest query x longest context) and
    # every value of the cache
    room = min(int(2.0e9) // (c["seqs"] * hq * max(c["q_hi"], c["q_long"])),
               int(3.0e8) // (c["seqs"] * hkv * d))
    c["ctx_hi"] = _log_int(rng, 64, max(65, min(32000, room)))
    c["ctx_lo"] = rng.choice((0, c["ctx_hi"] // 2))
    return c


def _lengths(case):
    """(tokens cached before, new tokens) of every sequence: the case's own, whatever the seed."""
    rng = random.Random(case["lens"])
    ctx, new = [], []
    for i in range(case["seqs"]):
        ctx.append(rng.randint(case["ctx_lo"], case["ctx_hi"]))
        long = case["long_every"] and i % case["long_every"] == 0
        new.append(rng.randint((case["q_long"] + 1) // 2, case["q_long"]) if long
                   else rng.randint(case["q_lo"], case["q_hi"]))
    return ctx, new


def _blocks(n):
    return (n + PAGE - 1) // PAGE


# --------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"step": _prepare_step, "extend": _prepare_extend, "score": _prepare_score}[
        case["op"]](case, gen)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32).to("cuda")


def _prepare_step(case, gen):
    ctx, new = _lengths(case)
    held = sum(_blocks(c) for c in ctx)
    wanted = sum(_blocks(c + n) - _blocks(c) for c, n in zip(ctx, new))
    ids = torch.randperm(held + wanted + 1000, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((case["seqs"], case["max_blocks"]), -1, dtype=torch.int32, device="cuda")
    first = _int32([_blocks(c) for c in ctx])[:, None]
    col = torch.arange(case["max_blocks"], device="cuda")[None]
    table[col < first] = ids[:held]
    total = sum(new)
    return dict(case=case, ctx=_int32(ctx), new=_int32(new), table=table,
                free=ids[held:].contiguous(), total=total,
                padded=(total + 255) // 256 * 256)  # steps are captured at padded token counts


def _group_codes(x, bits, asym):
    """Codes and the fp16 scale (and zero-point) of each group of 32 of the last dimension."""
    g = x.unflatten(-1, (-1, 32))
    if bits == 8:
        s = g.abs().amax(-1, keepdim=True) / 127
        return (torch.round(g / s).clamp(-128, 127).to(torch.int8).flatten(-2),
                s.squeeze(-1).half(), None)
    if asym:
        lo = g.amin(-1, keepdim=True)
        s = (g.amax(-1, keepdim=True) - lo).clamp_min(1e-8) / 15
        q, zero = torch.round((g - lo) / s).clamp(0, 15), lo.squeeze(-1).half()
    else:
        s = g.abs().amax(-1, keepdim=True) / 7
        q, zero = torch.round(g / s).clamp(-8, 7) + 8, None
    q = q.flatten(-2).to(torch.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), s.squeeze(-1).half(), zero


def _prepare_extend(case, gen):
    ctx, new = _lengths(case)
    lens = [c + n for c, n in zip(ctx, new)]
    hq, hkv, d, mode = case["hq"], case["hkv"], case["d"], case["mode"]
    dtype = DTYPES[case["q"]]
    pages = [_blocks(n) for n in lens]
    n_blocks = sum(pages)
    # keys: a few channels of every head ten times the others, with a mean of their own;
    # values: a mean per channel (what attention over a real cache averages)
    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")
    wide = torch.where(torch.rand(hkv, d, generator=gen, device="cuda") < 0.01, 10.0, 1.0)
    k_mean, v_mean = randn(hkv, d) * wide, randn(hkv, d)
    k = randn(n_blocks, PAGE, hkv, d) * wide * 0.5 + k_mean
    v = randn(n_blocks, PAGE, hkv, d) + v_mean
    s = dict(case=case, asym=mode == "int4_asym" or mode in ("k8v4", "kfpv4"))
    if mode.startswith("kfp"):
        s["k"], s["ks"], s["kz"] = k.to(dtype), None, None
    else:
        s["k"], s["ks"], s["kz"] = _group_codes(k, 8 if mode.startswith("k8") else 4, s["asym"])
    s["v"], s["vs"], s["vz"] = _group_codes(v, 8 if mode.endswith("v8") else 4, s["asym"])
    ids = torch.randperm(n_blocks, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(pages), dtype=torch.int32, device="cuda")
    col = torch.arange(max(pages), device="cuda")[None]
    table[col < _int32(pages)[:, None]] = ids
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return dict(s, query=randn(starts[-1], hq, d).to(dtype), table=table, lens=_int32(lens),
                starts=_int32(starts), max_len=max(lens), max_new=max(new))


def _prepare_score(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=gen, device="cuda") * 2.5
    ids = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    likely = torch.rand(rows, generator=gen, device="cuda") < 0.7
    x[torch.arange(rows, device="cuda"), ids] += torch.where(likely, 12.0, 0.0)
    if case["masked"]:
        off = torch.rand(rows, vocab, generator=gen, device="cuda") < case["masked"]
        off[torch.arange(rows, device="cuda"), ids] = False  # the token given was allowed
        x.masked_fill_(off, float("-inf"))
    return dict(case=case, logits=x.to(DTYPES[case["logits"]]), ids=ids)


# --------------------------------------------------------------------------- one pass
def run(state):
    return {"step": _run_step, "extend": _run_extend, "score": _run_score}[
        state["case"]["op"]](state)


def _run_step(s):
    if own:
        from knlp_b200 import cache
        t = cache.build_step(s["ctx"], s["new"], s["table"], s["free"], PAGE, s["padded"])
        return dict(query_start_loc=t.query_start_loc, seq_lens=t.seq_lens,
                    slot_mapping=t.slot_mapping, positions=t.positions,
                    blocks_taken=t.blocks_taken, block_table=s["table"])
    ctx, new, table, free = s["ctx"].long(), s["new"].long(), s["table"], s["free"]
    ends = torch.cumsum(new, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    lens = ctx + new
    first, last = (ctx + PAGE - 1) // PAGE, (lens + PAGE - 1) // PAGE
    taken = torch.cumsum(last - first, 0)
    col = torch.arange(table.shape[1], device="cuda")[None]
    source = (taken - (last - first) - first)[:, None] + col
    fresh = (col >= first[:, None]) & (col < last[:, None])
    table = torch.where(fresh, free[source.clamp(0, free.numel() - 1)], table)
    t = torch.arange(s["padded"], device="cuda")
    row = torch.searchsorted(ends, t, right=True)
    there = row < ends.numel()
    row = row.clamp_max(ends.numel() - 1)
    pos = torch.where(there, ctx[row] + t - starts[row], 0)
    slot = table[row, pos // PAGE].long() * PAGE + pos % PAGE
    return dict(query_start_loc=starts.int(), seq_lens=lens.int(),
                slot_mapping=torch.where(there, slot, -1), positions=pos,
                blocks_taken=taken[-1:].int(), block_table=table)


def _own_extend(s):
    from knlp_b200 import ops
    mode, more = s["case"]["mode"], {}
    call = {"int4_asym": ops.fused_int4_extend, "int4_sym": ops.fused_int4_extend,
            "k8v4": ops.kint8_vint4_extend, "k8v8": ops.kint8_vint8_extend,
            "kfpv4": ops.kfp16_vint4_extend, "kfpv8": ops.kfp16_vint8_extend}[mode]
    if not mode.endswith("v8"):
        more = dict(v_zeros=s["vz"], asymmetric=s["asym"])
    if mode.startswith("int4"):
        more["k_zeros"] = s["kz"]
    scales = (s["vs"],) if mode.startswith("kfp") else (s["ks"], s["vs"])
    return call(s["query"], s["k"], s["v"], *scales, s["table"], s["lens"], s["starts"],
                s["case"]["hkv"], s["case"]["d"], max_seq_len=s["max_len"],
                max_query_len=s["max_new"], **more)


def _values(codes, scales, zeros, table, d):
    """The cached rows of every sequence, [seqs, heads, tokens, d] in fp32."""
    c = codes[table].flatten(1, 2)
    if scales is None:
        return c.float().transpose(1, 2)
    sc = scales[table].flatten(1, 2).float()
    if c.dtype == torch.uint8:
        c = torch.stack([c & 15, c >> 4], dim=-1).flatten(-2).float()
        if zeros is None:
            c -= 8
    else:
        c = c.float()
    c = c.unflatten(-1, (-1, 32)).mul_(sc[..., None])
    if zeros is not None:
        c += zeros[table].flatten(1, 2).float()[..., None]
    return c.flatten(-2).transpose(1, 2)


def _run_extend(s):
    if own:
        return _own_extend(s)
    case, q, starts, lens = s["case"], s["query"], s["starts"].long(), s["lens"].long()
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    table, n, most = s["table"].long(), case["seqs"], s["max_new"]
    k = _values(s["k"], s["ks"], s["kz"], table, d)
    i = torch.arange(most, device="cuda")[None]
    at = (starts[:-1, None] + i).clamp_max(q.shape[0] - 1)  # rows behind a short one: any row
    qp = q[at].float().view(n, most, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(
        n, hkv, -1, d)
    score = torch.matmul(qp, k.transpose(2, 3)).mul_(d ** -0.5)
    del k
    score = score.view(n, hkv, hq // hkv, most, -1)
    limit = (lens - (starts[1:] - starts[:-1]))[:, None] + i  # position of each query token
    t = torch.arange(score.shape[-1], device="cuda")
    score.masked_fill_((t > limit[..., None])[:, None, None], float("-inf"))
    score -= score.amax(-1, keepdim=True)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    v = _values(s["v"], s["vs"], s["vz"], table, d)
    o = torch.matmul(score.view(n, hkv, -1, score.shape[-1]), v).view(n, hkv, hq // hkv, most, d)
    o = (o / total).permute(0, 3, 1, 2, 4).reshape(n, most, hq, d)
    r = torch.arange(q.shape[0], device="cuda")
    row = torch.searchsorted(starts[1:], r, right=True)
    return o[row, r - starts[row]].to(q.dtype)


def _run_score(s):
    case, logits, ids = s["case"], s["logits"], s["ids"]
    if own:
        from knlp_b200 import scoring
        r = scoring.token_logprobs(logits, ids, top_k=case["top"])
        return dict(logprob=r.logprob, entropy=r.entropy, rank=r.rank, top_ids=r.top_ids,
                    top_logprobs=r.top_logprobs)
    x = logits.float()
    m = x.amax(-1, keepdim=True)
    shifted = x - m
    p = shifted.exp()
    total = p.sum(-1, keepdim=True)
    log_total = total.log()
    weighted = torch.where(p > 0, p * shifted, 0).sum(-1, keepdim=True)
    given = x.gather(1, ids[:, None])
    # the k largest, lower index first among equals: one integer key of value and index
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -2147483648 - bits, bits) * (1 << 20)
    key += (1 << 20) - 1 - torch.arange(x.shape[1], device="cuda")
    top = (1 << 20) - 1 - (key.topk(case["top"], dim=-1).values & ((1 << 20) - 1))
    return dict(logprob=((given - m) - log_total)[:, 0],
                entropy=(log_total - weighted / total)[:, 0],
                rank=((x > given).sum(-1) + 1).int(), top_ids=top,
                top_logprobs=x.gather(1, top) - m - log_total)


# --------------------------------------------------------------------------- what it takes
def work(case):
    if case["op"] == "step":
        ctx, new = _lengths(case)
        total = sum(new)
        padded = (total + 255) // 256 * 256
        taken = sum(_blocks(c + n) - _blocks(c) for c, n in zip(ctx, new))
        # lengths in, offsets and lengths out; slot and position of every token; a block id
        # read and a table entry written for every block taken
        return {"bytes": 16 * case["seqs"] + 16 * padded + 8 * taken, "flops": 0}
    if case["op"] == "score":
        size = 4 if case["logits"] == "f32" else 2
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (8 + 12 + 12 * case["top"]), "flops": 4 * n}
    ctx, new = _lengths(case)
    hq, hkv, d, mode = case["hq"], case["hkv"], case["d"], case["mode"]
    groups = d // 32
    asym = mode == "int4_asym" or mode in ("k8v4", "kfpv4")
    four = d // 2 + groups * (4 if asym else 2)
    eight = d + 2 * groups
    row = {"int4": four, "k8v4": eight, "k8v8": eight, "kfpv": 2 * d}[mode[:4]]
    row += eight if mode.endswith("v8") else four
    tokens = sum(c + n for c, n in zip(ctx, new))
    seen = sum(c * n + n * (n + 1) // 2 for c, n in zip(ctx, new))  # (query, key) pairs
    return {"bytes": tokens * hkv * row + 4 * sum(new) * hq * d + 4 * (tokens // PAGE),
            "flops": 4 * seen * hq * d}


# --------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["op"] == "step":
        return None  # whole numbers
    state = prepare(case, seed)
    return _exact_score(state) if case["op"] == "score" else _exact_extend(state)


def _exact_score(s):
    logits, ids, top = s["logits"], s["ids"].tolist(), s["case"]["top"]
    out = {"logprob": [], "entropy": [], "rank": None, "top_ids": None, "top_logprobs": []}
    for r in range(logits.shape[0]):
        lp = logits[r].double()
        lp = lp - torch.logsumexp(lp, 0)
        out["logprob"].append(lp[ids[r]])
        out["entropy"].append(-torch.special.xlogy(lp.exp(), lp.exp()).sum())
        out["top_logprobs"].append(torch.sort(lp, descending=True).values[:top])
    return {k: None if v is None else torch.stack(v) for k, v in out.items()}


def _exact_rows(codes, scales, zeros, blocks, head, n):
    c = codes[blocks, :, head].reshape(blocks.numel() * PAGE, -1)[:n]
    if scales is None:
        return c.double()
    if c.dtype == torch.uint8:
        wide = torch.empty(n, 2 * c.shape[1], dtype=torch.float64, device="cuda")
        wide[:, 0::2], wide[:, 1::2] = (c % 16).double(), (c // 16).double()
        c = wide - 8 if zeros is None else wide
    group = torch.arange(c.shape[1], device="cuda") // 32
    flat = lambda a: a[blocks, :, head].reshape(blocks.numel() * PAGE, -1)[:n].double()[:, group]
    c = c.double() * flat(scales)
    return c if zeros is None else c + flat(zeros)


def _exact_extend(s):
    hq, hkv, d = s["case"]["hq"], s["case"]["hkv"], s["case"]["d"]
    starts, lens, rep = s["starts"].tolist(), s["lens"].tolist(), hq // hkv
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        blocks = s["table"][i, :_blocks(n)].long()
        for h in range(hkv):
            k = _exact_rows(s["k"], s["ks"], s["kz"], blocks, h, n)
            v = _exact_rows(s["v"], s["vs"], s["vz"], blocks, h, n)
            for c in range(a, b, 1024):  # query rows at a time
                e = min(b, c + 1024)
                q = s["query"][c:e, h * rep:(h + 1) * rep].double()
                w = torch.einsum("thd,kd->htk", q, k) / math.sqrt(d)
                seen = torch.arange(n, device="cuda")[None] <= (
                    n - (b - torch.arange(c, e, device="cuda")))[:, None]
                w = torch.softmax(w.masked_fill(~seen, -math.inf), -1)
                out[c:e, h * rep:(h + 1) * rep] = torch.einsum("htk,kd->thd", w, v)
    return out
