"""More operators of the paged 8-bit KV cache (``megakernel_amd.kv8``), as
cases that can be timed and compared: rotary positions in both layouts, for
part of a head and scaled for long contexts; attention whose scores are capped
by a tanh or biased by distance and whose rows see a window, a document or a
prefix; the attention weight that each cached position gathers; and the
eviction of the positions that gathered least.

Shapes are those of this repository's presets (16 query / 8 KV heads of 64 or
128) and of its tests and benchmark (contexts of 512 to 32,768 positions, 16
sequences at once, prompts of 1,024 tokens); odd lengths are among them.

Kinds:
  rotary  the rotation of every q and k head by its token's position
  attend  attention of each sequence's newest tokens over its blocks: the
          score of row p and position j is cap * tanh(scale * q.k / cap)
          - slope[head] * |p - j|, and the row sees max(first, p + 1 - window)
          <= j < max(p + 1, prefix)
  weigh   the same, with each row's log-sum-exp, and the weights that each
          position got, summed over rows and the heads that share a KV head,
          added to what it had (positions of the new rows start at zero)
  evict   of each sequence and KV head the heaviest positions are chosen, with
          the first and the newest ones, and moved into blocks of their own,
          which are then read back
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

THETA = 1e6
BLOCKS = (16, 32, 64, 128)
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
ATTEND = dict(cap=0.0, slopes=False, window=0, doc_lo=0, doc_hi=0, prefix=0)


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of 16 sequences: the launch itself is what counts
        dict(name="rotary step", kind="rotary", tokens=16, n_q=16, n_kv=8, dim=64, turned=64, interleaved=True,
             scaling="none", src="bf16", dst="bf16", first=4000),
        # prompts at far positions of a context four times as long as trained for, half of each head turned
        dict(name="rotary prompt", kind="rotary", tokens=8192, n_q=16, n_kv=8, dim=128, turned=64, interleaved=False,
             scaling="parts", src="bf16", dst="bf16", first=24576),
        # whole heads, neighbours as pairs, from the QKV product's fp32
        dict(name="rotary wide", kind="rotary", tokens=4096, n_q=16, n_kv=8, dim=128, turned=128, interleaved=True,
             scaling="linear", src="fp32", dst="bf16", first=0),
        # batched decode with capped scores
        dict(ATTEND, name="decode capped", kind="attend", n_q=16, n_kv=8, dim=64, block=32, seqs=16, new_lo=1, new_hi=1,
             ctx_lo=512, ctx_hi=4096, cap=50.0),
        # a layer with a window, deep into a long context
        dict(ATTEND, name="decode window", kind="attend", n_q=16, n_kv=8, dim=128, block=64, seqs=1, new_lo=1, new_hi=1,
             ctx_lo=32768, ctx_hi=32768, window=4096),
        # drafted tokens of every sequence with a bias by distance
        dict(ATTEND, name="verify biased", kind="attend", n_q=16, n_kv=8, dim=128, block=16, seqs=16, new_lo=3, new_hi=6,
             ctx_lo=700, ctx_hi=8191, slopes=True),
        # passages of 100 to 700 tokens packed into one row, none of which sees another
        dict(ATTEND, name="prompt documents", kind="attend", n_q=16, n_kv=8, dim=64, block=32, seqs=1, new_lo=4096,
             new_hi=4096, ctx_lo=4096, ctx_hi=4096, doc_lo=101, doc_hi=701),
        # the last 1,024 tokens of a long prompt, capped and after a prefix that sees itself whole
        dict(ATTEND, name="prompt at depth", kind="attend", n_q=16, n_kv=8, dim=128, block=64, seqs=1, new_lo=1024,
             new_hi=1024, ctx_lo=16384, ctx_hi=16384, cap=30.0, prefix=96),
        # a decode step that keeps count of what its positions are worth
        dict(ATTEND, name="weigh step", kind="weigh", n_q=16, n_kv=8, dim=64, block=32, seqs=16, new_lo=1, new_hi=1,
             ctx_lo=512, ctx_hi=4096),
        # the same for ragged prompts
        dict(ATTEND, name="weigh prompts", kind="weigh", n_q=16, n_kv=8, dim=128, block=32, seqs=4, new_lo=257,
             new_hi=2048, ctx_lo=1025, ctx_hi=6000, cap=50.0),
        # a long conversation cut down to an eighth
        dict(name="evict long", kind="evict", n_kv=8, dim=128, block=64, seqs=1, ctx_lo=32768, ctx_hi=32768, keep=4096,
             recent=512, sinks=4),
        # a full batch cut down to at most 1,000 positions each
        dict(name="evict batch", kind="evict", n_kv=8, dim=64, block=32, seqs=16, ctx_lo=512, ctx_hi=4096, keep=1000,
             recent=128, sinks=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "attend", "attend", "attend", "weigh", "evict"])
    n_kv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    while n_kv * group > 16:
        group -= 1
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128])
        turned = rng.choice([dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)])
        return dict(kind=kind, tokens=_log(rng, 1, 8192), n_q=n_kv * group, n_kv=n_kv, dim=dim, turned=turned,
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "base", "parts"]),
                    src=rng.choice(list(TYPES)), dst=rng.choice(list(TYPES)), first=_log(rng, 1, 100000) - 1)
    dim, block, seqs = rng.choice([64, 128]), rng.choice(BLOCKS), rng.randint(1, 16)
    ctx_hi = _log(rng, 1, 32768 // seqs)
    ctx_lo = _log(rng, 1, ctx_hi)
    if kind == "evict":
        keep = _log(rng, 1, max(1, min(ctx_hi, 4096)))
        recent = rng.randint(0, keep)
        return dict(kind=kind, n_kv=n_kv, dim=dim, block=block, seqs=seqs, ctx_lo=ctx_lo, ctx_hi=ctx_hi, keep=keep,
                    recent=recent, sinks=rng.randint(0, min(8, keep - recent)))
    new_hi = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(ctx_hi, 2048)))
    while seqs * new_hi * ctx_hi * n_kv * group > 2 ** 28 and new_hi > 1:
        new_hi = max(1, new_hi // 2)
    case = dict(ATTEND, kind=kind, n_q=n_kv * group, n_kv=n_kv, dim=dim, block=block, seqs=seqs,
                new_lo=rng.randint(1, new_hi), new_hi=new_hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi)
    if rng.random() < 0.4:
        case["cap"] = rng.uniform(5.0, 60.0)
    if rng.random() < 0.3:
        case["slopes"] = True
    if rng.random() < 0.3:
        case["window"] = _log(rng, 1, ctx_hi)
    if rng.random() < 0.3:
        case["doc_hi"] = _log(rng, 1, ctx_hi)
        case["doc_lo"] = rng.randint(1, case["doc_hi"])
    if rng.random() < 0.3:
        case["prefix"] = rng.randint(1, 100)
    return case


def _spread(lo, hi, n, step):
    """n lengths from lo to hi, evenly apart, in an order that `step` mixes."""
    return [lo + (hi - lo) * ((i * step) % n) // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """(context, new tokens) of each sequence; the context includes the new tokens."""
    n = case["seqs"]
    ctx = _spread(case["ctx_lo"], case["ctx_hi"], n, 1)
    if case["kind"] == "evict":
        return ctx, ctx
    return ctx, [min(a, b) for a, b in zip(_spread(case["new_lo"], case["new_hi"], n, 1), ctx)]


def _doc_starts(case, ctx):
    """Where the document of each position of one sequence begins."""
    if not case["doc_hi"]:
        return np.zeros(ctx, np.int64)
    out, at, i, sizes = np.empty(ctx, np.int64), 0, 0, _spread(case["doc_lo"], case["doc_hi"], 7, 3)
    while at < ctx:
        out[at : at + sizes[i % 7]] = at
        at, i = at + sizes[i % 7], i + 1
    return out


def _seen(case):
    """The positions [lo, hi) that each new row of each sequence sees."""
    out = []
    for c, n in zip(*_lengths(case)):
        p = np.arange(c - n, c)
        lo = _doc_starts(case, c)[p]
        if case["window"]:
            lo = np.maximum(lo, p + 1 - case["window"])
        out.append((lo, np.maximum(p + 1, c * case["prefix"] // 100)))
    return out


def _size(name):
    return {"bf16": 2, "fp32": 4}[name]


def work(case):
    if case["kind"] == "rotary":
        n = case["tokens"] * (case["n_q"] + case["n_kv"])
        return {"bytes": n * case["dim"] * (_size(case["src"]) + _size(case["dst"])) + 4 * case["tokens"],
                "flops": 3 * n * case["turned"]}
    ctx, new = _lengths(case)
    row, n_kv = case["n_kv"] * case["dim"], case["n_kv"]
    if case["kind"] == "evict":
        kept = sum(min(c, case["keep"]) for c in ctx)
        # the weights of every position; of kept ones the number and the weight,
        # the codes read and written, then read again and written as bf16
        return {"bytes": n_kv * (4 * sum(ctx) + 8 * kept) + 2 * row * kept * (1 + 1 + 1 + 2), "flops": 4 * row * kept}
    seen = pairs = 0
    for (lo, hi), c in zip(_seen(case), ctx):
        edge = np.zeros(c + 1, np.int64)
        np.add.at(edge, lo, 1)
        np.add.at(edge, hi, -1)
        seen += int((np.cumsum(edge) > 0).sum())
        pairs += int((hi - lo).sum())
    w = {"bytes": 2 * row * seen + 4 * case["n_q"] * case["dim"] * sum(new) + 8 * n_kv * (seen // case["block"]),
         "flops": 4 * case["n_q"] * case["dim"] * pairs}
    if case["kind"] == "weigh":
        w["bytes"] += 4 * case["n_q"] * sum(new) + 8 * n_kv * seen
        w["flops"] += case["n_q"] * pairs
    return w


# ------------------------------------------------------------------ inputs
class State:
    pass


def _rows(shape, gen, spread):
    """Rows of K or V: dimensions of unlike size, as norms' gains and weights leave them, and a few large ones."""
    dim = shape[-1]
    size = torch.exp(0.5 * torch.randn(dim, generator=gen, device="cuda"))
    size[torch.randint(0, dim, (2,), generator=gen, device="cuda")] *= 6.0
    return torch.randn(shape, generator=gen, device="cuda") * size * spread


def _tables(lens, block, gen, ids=None):
    """Block tables of sequences of these lengths, dealt at random, and the blocks left over."""
    n, width = len(lens), max(-(-c // block) for c in lens)
    used = sum(-(-c // block) for c in lens)
    if ids is None:
        ids = torch.randperm(used + 3, generator=gen, device="cuda").to(torch.int32).cpu()
    table, at = torch.full((n, width), -1, dtype=torch.int32), 0
    for i, c in enumerate(lens):
        k = -(-c // block)
        table[i, :k] = ids[at : at + k]
        at += k
    return table, ids[at:]


def _starts(new):
    return torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32).cuda()


def _filled(s, n_kv, dim, block, gen):
    """Pools that hold quantised rows in every block."""
    k = _rows((s.n_blocks, n_kv, block, dim), gen, 1.0)
    v = _rows((s.n_blocks, n_kv, block, dim), gen, 0.4)
    s.k_scale, s.v_scale = _scale_of(k.abs().amax((2, 3))), _scale_of(v.abs().amax((2, 3)))
    s.k = _encode(k / s.k_scale[:, :, None, None]).view(torch.uint8)
    s.v = _encode(v / s.v_scale[:, :, None, None]).view(torch.uint8).transpose(2, 3).contiguous()


def _frequencies(turned, scaling):
    """Inverse frequencies of `turned` dimensions for a context four times as long as 8,192."""
    factor, original = 4.0, 8192
    base = THETA * factor ** (turned / (turned - 2)) if scaling == "base" and turned > 2 else THETA
    inv = np.array([base ** (-2.0 * i / turned) for i in range(turned // 2)])
    if scaling == "linear":
        inv = inv / factor
    if scaling == "parts":  # few turns within the original context: as linear; many: as they are; a ramp between
        turns = original * inv / (2 * math.pi)
        stay = np.clip((turns - 1) / (32 - 1), 0, 1)
        inv = inv * stay + inv / factor * (1 - stay)
    return torch.from_numpy(inv.astype(np.float32)).cuda(), 0.1 * math.log(factor) + 1 if scaling == "parts" else 1.0


def _weights(n, n_kv, width, gen):
    """Gathered weights: a long tail, some positions that never got any, the first ones heavy."""
    w = torch.exp(2 * torch.randn((n, n_kv, width), generator=gen, device="cuda"))
    w *= torch.rand((n, n_kv, width), generator=gen, device="cuda") > 0.2
    w[:, :, :4] += 100.0
    return w


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = State()
    s.case = case
    kind, dim, n_kv = case["kind"], case["dim"], case["n_kv"]
    if kind == "rotary":
        t, n_q = case["tokens"], case["n_q"]
        s.qkv = torch.randn((t, n_q + 2 * n_kv, dim), generator=gen, device="cuda").mul_(2.0).to(TYPES[case["src"]])
        s.q, s.rows_k = s.qkv[:, :n_q], s.qkv[:, n_q : n_q + n_kv]
        s.inv_freq, s.amplitude = _frequencies(case["turned"], case["scaling"])
        s.pos = torch.arange(case["first"], case["first"] + t, dtype=torch.int32, device="cuda")
        s.q_out = torch.empty((t, n_q, dim), dtype=TYPES[case["dst"]], device="cuda")
        s.k_out = torch.empty((t, n_kv, dim), dtype=TYPES[case["dst"]], device="cuda")
        return s
    lens, new = _lengths(case)
    block, n = case["block"], case["seqs"]
    table, left = _tables(lens, block, gen)
    s.n_blocks = int(table.max()) + 1 if not len(left) else max(int(table.max()), int(left.max())) + 1
    if kind == "evict":
        s.kept_lens = [min(c, case["keep"]) for c in lens]
        extra = sum(-(-c // block) for c in s.kept_lens)
        more = torch.randperm(extra, generator=gen, device="cuda").to(torch.int32).cpu() + s.n_blocks
        s.new_table = _tables(s.kept_lens, block, gen, more)[0].cuda()
        s.n_blocks += extra
    s.table = table.cuda()
    s.q_start, s.kv_len = _starts(new), torch.tensor(lens, dtype=torch.int32).cuda()
    s.tokens, s.max_kv, s.max_new = int(sum(new)), int(max(lens)), int(max(new))
    _filled(s, n_kv, dim, block, gen)
    if kind in ("weigh", "evict"):
        s.mass = _weights(n, n_kv, s.table.shape[1] * block, gen)
    if own:
        from megakernel_amd import kv8

        s.cache = kv8.Cache(s.k, s.v, s.k_scale, s.v_scale)
        s.batch = kv8.Batch(s.table, s.q_start, s.kv_len, s.tokens, s.max_kv)
    if kind == "evict":
        s.kept = torch.empty((n, n_kv, case["keep"]), dtype=torch.int32, device="cuda")
        s.kept_len = torch.empty(n, dtype=torch.int32, device="cuda")
        s.new_mass = torch.zeros((n, n_kv, s.new_table.shape[1] * block), device="cuda")
        s.back_start, s.back_tokens = _starts(s.kept_lens), int(sum(s.kept_lens))
        s.k_out = torch.empty((s.back_tokens, n_kv, dim), dtype=torch.bfloat16, device="cuda")
        s.v_out = torch.empty_like(s.k_out)
        if own:
            s.back = kv8.Batch(s.new_table, s.back_start, s.kept_len, s.back_tokens, max(s.kept_lens))
        return s
    n_q = case["n_q"]
    s.q = (torch.randn((s.tokens, n_q, dim), generator=gen, device="cuda") * 1.5).to(torch.bfloat16)
    s.out = torch.empty_like(s.q)
    s.lse = torch.empty((s.tokens, n_q), device="cuda")
    s.slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / n_q) for h in range(n_q)]).cuda() if case["slopes"] else None
    s.first = s.prefix = None
    if case["doc_hi"]:
        s.first = torch.from_numpy(np.concatenate([_doc_starts(case, c)[c - m :] for c, m in zip(lens, new)]).astype(np.int32)).cuda()
    if case["prefix"]:
        s.prefix = torch.tensor([c * case["prefix"] // 100 for c in lens], dtype=torch.int32).cuda()
    if own:
        s.scores = kv8.Scores(softcap=case["cap"], slopes=s.slopes, window=case["window"], first=s.first, prefix=s.prefix)
    return s


# -------------------------------------------------------------- plain form
def _scale_of(amax):
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    m, e = torch.frexp(amax.float())  # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e - 9 + (m > 0.875), -126).clamp_min(-126)
    return torch.exp2(e.double()).float()


def _encode(x):
    """e4m3 of values of at most 448: nearest, ties to even."""
    return x.to(torch.float8_e4m3fn)


def _values(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _places(q_start, kv_len, tokens):
    """(sequence, position) of each row."""
    t = torch.arange(tokens, device=q_start.device)
    seq = torch.searchsorted(q_start[1:].long().contiguous(), t, right=True)
    return seq, (kv_len[seq] - q_start[seq + 1] + t).long()


def _plain_rotary(s):
    turned = s.case["turned"]
    angle = s.pos.double()[:, None] * s.inv_freq.double()  # 32 bits lose far positions' angles
    c, sn = (f.float()[:, None] * s.amplitude for f in (angle.cos(), angle.sin()))

    def turn(x, dtype):
        x = x.float()
        part, rest = x[..., :turned], x[..., turned:]
        if s.case["interleaved"]:
            a, b = part[..., 0::2], part[..., 1::2]
            part = torch.stack((a * c - b * sn, b * c + a * sn), -1).flatten(-2)
        else:
            a, b = part.chunk(2, -1)
            part = torch.cat((a * c - b * sn, b * c + a * sn), -1)
        return torch.cat((part, rest), -1).to(dtype)

    return [turn(s.q, s.q_out.dtype), turn(s.rows_k, s.k_out.dtype)]


def _plain_attend(s):
    """Output, log-sum-exp and each position's weight of this pass."""
    case = s.case
    n, block, dim, n_kv = s.kv_len.shape[0], s.k.shape[2], case["dim"], case["n_kv"]
    group, width = case["n_q"] // n_kv, s.table.shape[1]
    blk = s.table.clamp_min(0).long()
    k = _values(s.k[blk]) * s.k_scale[blk][..., None, None]  # [n, width, n_kv, block, dim]
    v = _values(s.v[blk]) * s.v_scale[blk][..., None, None]  # [n, width, n_kv, dim, block]
    k = k.permute(0, 2, 4, 1, 3).reshape(n * n_kv, dim, width * block).contiguous()
    v = v.permute(0, 2, 1, 4, 3).reshape(n * n_kv, width * block, dim).contiguous()
    seq, pos = _places(s.q_start, s.kv_len, s.tokens)
    at = torch.arange(s.tokens, device=seq.device) - s.q_start[seq]
    q = torch.zeros((n, s.max_new, n_kv, group, dim), device="cuda")
    q[seq, at] = s.q.float().view(-1, n_kv, group, dim)
    lo, hi = torch.zeros_like(pos), pos + 1
    if s.first is not None:
        lo = torch.maximum(lo, s.first.long())
    if case["window"]:
        lo = torch.maximum(lo, pos + 1 - case["window"])
    if s.prefix is not None:
        hi = torch.maximum(hi, s.prefix.long()[seq])
    spans = []
    for x in (lo, hi, pos):  # nothing is seen by rows that are not there
        y = torch.zeros((n, s.max_new), device="cuda", dtype=torch.long)
        y[seq, at] = x
        spans.append(y[:, :, None])
    j = torch.arange(width * block, device="cuda")
    hidden = (j < spans[0]) | (j >= spans[1])
    q = q.permute(0, 2, 1, 3, 4).reshape(n * n_kv, s.max_new * group, dim)
    x = torch.bmm(q * (1 / math.sqrt(dim)), k).view(n, n_kv, s.max_new, group, width * block)
    if case["cap"]:
        x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
    if s.slopes is not None:
        far = (j - spans[2]).abs().float()
        x -= s.slopes.view(n_kv, 1, group, 1) * far[:, None, :, None]
    x.masked_fill_(hidden[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min(-1e30)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    x = x / total.clamp_min(1e-30)
    o = torch.bmm(x.view(n * n_kv, s.max_new * group, width * block), v).view(n, n_kv, s.max_new, group, dim)
    out = o.permute(0, 2, 1, 3, 4)[seq, at].reshape(s.tokens, case["n_q"], dim).to(torch.bfloat16)
    if case["kind"] == "attend":
        return out, None, None
    lse = (top + total.log())[..., 0].permute(0, 2, 1, 3)[seq, at].reshape(s.tokens, case["n_q"])
    return out, lse, x.sum((2, 3))


def _plain_weigh(s):
    out, lse, got = _plain_attend(s)
    j = torch.arange(s.mass.shape[2], device="cuda")
    rows = (s.q_start[1:] - s.q_start[:-1])[:, None]
    older, there = j < s.kv_len[:, None] - rows, j < s.kv_len[:, None]
    was = torch.where(older[:, None], s.mass, 0.0)
    s.mass.copy_(torch.where(there[:, None], was + got, s.mass))
    return [out, lse, s.mass]


def _plain_evict(s):
    case, block = s.case, s.case["block"]
    n, keep = s.kv_len.shape[0], case["keep"]
    j = torch.arange(s.mass.shape[2], device="cuda")
    there, always = j < s.kv_len[:, None], (j >= s.kv_len[:, None] - case["recent"]) | (j < case["sinks"])
    key = torch.where(always[:, None], math.inf, s.mass)
    key = torch.where(there[:, None], key, -1.0)
    best = key.sort(dim=-1, descending=True, stable=True).indices[:, :, :keep]
    if best.shape[2] < keep:
        best = torch.cat((best, best.new_zeros(best.shape[:2] + (keep - best.shape[2],))), -1)
    s.kept_len.copy_(s.kv_len.clamp_max(keep))
    real = torch.arange(keep, device="cuda") < s.kept_len[:, None]
    best = torch.where(real[:, None], best, s.mass.shape[2]).sort(-1).values
    s.kept.copy_(torch.where(real[:, None], best, -1))
    # the rows of every new block, quantised anew
    seq, place = _places(s.back_start, s.kept_len, s.back_tokens)
    src = s.kept[seq, :, place].long()  # [tokens][n_kv]
    heads = torch.arange(case["n_kv"], device="cuda")
    s.new_mass[seq, :, place] = s.mass[seq[:, None], heads, src]
    old, row = s.table[seq[:, None], src // block].long(), src % block
    blk, to = s.new_table[seq, place // block].long(), place % block
    k = _values(s.k[old, heads, row]) * s.k_scale[old, heads][..., None]
    v = _values(s.v[old, heads, :, row]) * s.v_scale[old, heads][..., None]
    outs = []
    for x, codes, scale, rows_first in ((k, s.k, s.k_scale, True), (v, s.v, s.v_scale, False)):
        most = torch.zeros_like(scale).index_reduce_(0, blk, x.abs().amax(-1), "amax")
        scale[blk] = _scale_of(most)[blk]
        fresh = _encode(x / scale[blk][..., None])
        if rows_first:
            codes[blk, :, to] = fresh.view(torch.uint8)
        else:
            codes[blk, :, :, to] = fresh.view(torch.uint8)
        outs.append((fresh.float() * scale[blk][..., None]).to(torch.bfloat16))
    return [s.kept, s.kept_len, s.new_mass, *outs, s.k_scale, s.v_scale]


# ---------------------------------------------------------------- one pass
def run(s):
    case = s.case
    kind = case["kind"]
    if own:
        from megakernel_amd import kv8

        if kind == "rotary":
            kv8.rotary(s.q, s.rows_k, s.inv_freq, s.pos, s.q_out, s.k_out, interleaved=case["interleaved"],
                       amplitude=s.amplitude)
            return [s.q_out, s.k_out]
        if kind == "attend":
            kv8.attention(s.cache, s.batch, s.q, s.out, scores=s.scores)
            return [s.out]
        if kind == "weigh":
            kv8.attention(s.cache, s.batch, s.q, s.out, scores=s.scores, lse=s.lse)
            kv8.weigh(s.cache, s.batch, s.q, s.lse, s.mass, scores=s.scores)
            return [s.out, s.lse, s.mass]
        kv8.select(s.cache, s.batch, s.mass, s.kept, s.kept_len, recent=case["recent"], sinks=case["sinks"])
        kv8.compact(s.cache, s.batch, s.kept, s.kept_len, s.new_table, s.mass, s.new_mass)
        kv8.read(s.cache, s.back, s.k_out, s.v_out)
        return [s.kept, s.kept_len, s.new_mass, s.k_out, s.v_out, s.k_scale, s.v_scale]
    if kind == "rotary":
        return _plain_rotary(s)
    if kind == "attend":
        return [_plain_attend(s)[0]]
    return _plain_weigh(s) if kind == "weigh" else _plain_evict(s)


# ---------------------------------------------------------------- 64 bits
_TABLE = [((c & 7) * 2.0 ** -9 if not c >> 3 & 15 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3 & 15) - 7)) * (-1) ** (c >> 7)
          for c in range(256)]


def _exact_values(codes):
    return torch.tensor(_TABLE, dtype=torch.float64, device="cuda")[codes.long()]


def _exact_round(x):
    """The e4m3 value nearest to x, ties to the even mantissa."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -20))).clamp_min(-6)
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_rotary(s, case):
    out, turned = [], case["turned"]
    for x in (s.q, s.rows_k):
        y = x.double().clone()
        first = slice(0, turned, 2) if case["interleaved"] else slice(0, turned // 2)
        second = slice(1, turned, 2) if case["interleaved"] else slice(turned // 2, turned)
        size = torch.tensor(float(np.float32(s.amplitude)), dtype=torch.float64, device="cuda")
        z = torch.complex(y[..., first], y[..., second]) * torch.polar(size, s.pos.double()[:, None, None] * s.inv_freq.double())
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return out


def _exact_evict(s, case, k, v, table, lens):
    block, n_kv, keep = case["block"], case["n_kv"], case["keep"]
    kept = np.full((len(lens), n_kv, keep), -1, np.int64)
    mass, new_mass = s.mass.double().cpu().numpy(), s.new_mass.double().cpu().numpy().copy()
    k_scale, v_scale = s.k_scale.double(), s.v_scale.double()
    new_table, outs = s.new_table.tolist(), []
    for i, c in enumerate(lens):
        m, both = min(c, keep), []
        for h in range(n_kv):
            fixed = set(range(min(case["sinks"], c))) | set(range(max(0, c - case["recent"]), c))
            # by falling weight, then by rising position
            order = sorted((j for j in range(c) if j not in fixed), key=lambda j: (-mass[i, h, j], j))
            kept[i, h, :m] = sorted((sorted(fixed) + order)[:m])
            new_mass[i, h, :m] = mass[i, h, kept[i, h, :m]]
            src = torch.from_numpy(kept[i, h, :m]).cuda()
            ids = torch.tensor(table[i], device="cuda")[src // block]
            both.append((k[ids, h, src % block], v[ids, h, src % block]))
        got = [torch.stack([b[z] for b in both], 1) for z in range(2)]  # [m][n_kv][dim]
        for j in range(-(-m // block)):
            to = new_table[i][j]
            for x, scale in zip(got, (k_scale, v_scale)):
                rows = x[j * block : (j + 1) * block]
                for h, most in enumerate(rows.abs().amax((0, 2)).tolist()):
                    scale[to, h] = 2.0 ** max(-126, math.ceil(math.log2(most / 448))) if most else 2.0 ** -126
                f = scale[to][None, :, None]
                rows.copy_(_exact_round(rows / f) * f)
        outs.append(got)
    kv = [torch.cat(x) for x in zip(*outs)]
    as_is = lambda x: torch.from_numpy(x).cuda()
    return [as_is(kept), torch.tensor([min(c, keep) for c in lens], device="cuda"), as_is(new_mass), *kv, k_scale, v_scale]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(s, case)
    lens, new = _lengths(case)
    dim, n_kv, block = case["dim"], case["n_kv"], case["block"]
    k = _exact_values(s.k) * s.k_scale.double()[:, :, None, None]
    v = _exact_values(s.v).transpose(2, 3) * s.v_scale.double()[:, :, None, None]
    table = s.table.tolist()
    if case["kind"] == "evict":
        return _exact_evict(s, case, k, v, table, lens)
    at, outs, lses = 0, [], []
    mass = s.mass.double() if case["kind"] == "weigh" else None
    for i, c in enumerate(lens):
        ids = torch.tensor(table[i][: -(-c // block)], device="cuda")
        ki, vi = (x[ids].transpose(0, 1).reshape(n_kv, -1, dim)[:, :c] for x in (k, v))
        q = s.q[at : at + new[i]].double()
        group, o = case["n_q"] // n_kv, torch.empty_like(q)
        lse = torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
        j, p = torch.arange(c, device="cuda"), torch.arange(c - new[i], c, device="cuda")[:, None]
        seen = j <= p
        if case["prefix"]:
            seen = seen | (j < c * case["prefix"] // 100)
        if case["window"]:
            seen = seen & (j > p - case["window"])
        if case["doc_hi"]:
            seen = seen & (j >= torch.from_numpy(_doc_starts(case, c)[c - new[i] :]).cuda()[:, None])
        if mass is not None:
            mass[i, :, c - new[i] : c] = 0
        for h in range(case["n_q"]):
            x = q[:, h] @ ki[h // group].T / math.sqrt(dim)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["slopes"]:
                x = x - s.slopes[h].double() * (p - j).abs()
            x = x.masked_fill(~seen, -math.inf)
            lse[:, h] = torch.logsumexp(x, -1)
            x = torch.exp(x - lse[:, h : h + 1])
            o[:, h] = x @ vi[h // group]
            if mass is not None:
                mass[i, h // group, :c] += x.sum(0)
        outs.append(o)
        lses.append(lse)
        at += new[i]
    return [torch.cat(outs)] if mass is None else [torch.cat(outs), torch.cat(lses), mass]
