"""The serving operators of the paged path, as cases that can be timed and checked.

Three operators of one serving step over a paged KV cache: the rotary embedding that appends
new tokens to the cache and keeps the gate's block means, the choice of kept blocks from gate
scores, and the attention of a chunk of new tokens over the cache. ``run`` computes each in its
plain form (elementary torch operations) or, with ``own`` set, through ``tasft_b200``.

A batch is packed along the token axis: sequence b has the new tokens
``cu_seqlens[b]:cu_seqlens[b+1]``, the last of its ``kv_len[b]`` tokens. Blocks are 64 tokens;
row i of a sequence's lists stands for the i-th 64-token block that its new tokens touch.
"""
import math
import random

import torch

own = False

BLOCK = 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


# ----------------------------------------------------------------------------- the cases
def listed():
    attend = dict(op="attend", hq=32, hk=8, dim=128, dtype="bf16", page=16, keep=0, per_head=False)
    append = dict(op="append", hq=32, hk=8, dim=128, dtype="bf16", page=16, rot=128, mixed=False, scaling="none",
                  base=500000.0)
    choose = dict(op="choose", hq=32, hk=8, floor=False)
    return [
        # one request in a chat: the next token, every cached block (latency counts)
        dict(attend, name="attend one token", seqs=1, longs=0, chunk=1, context=4000, shape=1),
        # the decode batch of the benchmark (64 sequences, 8192 tokens, 26 kept blocks), lengths as they come
        dict(attend, name="attend tokens of a batch", seqs=64, longs=0, chunk=1, context=8100, keep=26, shape=2),
        # a scheduler's step: two prompts being filled in beside 32 running requests
        dict(attend, name="attend a mixed step", seqs=34, longs=2, chunk=509, context=6000, keep=24, page=32, shape=3),
        # a chunk of a long prompt over everything before it, no blocks left out
        dict(attend, name="attend a chunk, all blocks", seqs=1, longs=1, chunk=2048, context=16384, page=64, shape=4),
        # the last chunk of the 32768-token prompt at 90% block sparsity, seven query heads to a KV head
        dict(attend, name="attend a chunk, kept blocks", seqs=1, longs=1, chunk=4096, context=28672, hq=28, hk=4,
             keep=51, page=64, shape=5),
        # a small model with a list for every query head, odd lengths, half precision
        dict(attend, name="attend lists per head", seqs=5, longs=5, chunk=333, context=1500, hq=8, hk=8, dim=64,
             dtype="f16", keep=7, per_head=True, page=128, shape=6),
        # the tokens of a decode batch enter the cache
        dict(append, name="append tokens of a batch", seqs=64, longs=0, chunk=1, context=2500, scaling="llama3",
             shape=7),
        # prompts enter the cache in large chunks, positions stretched fourfold
        dict(append, name="append chunks", seqs=4, longs=4, chunk=2048, context=30000, hq=28, hk=4, page=64,
             scaling="yarn", base=1000000.0, shape=8),
        # part of the head is rotated, in interleaved pairs; ragged chunks in half precision
        dict(append, name="append part of a head", seqs=7, longs=7, chunk=301, context=700, hq=8, hk=8, dim=64,
             dtype="f16", rot=32, mixed=True, page=32, scaling="linear", base=10000.0, shape=9),
        # kept blocks of a decode batch
        dict(choose, name="choose for a batch", seqs=64, longs=0, chunk=1, context=8100, keep=26, shape=10),
        # kept blocks of a chunk at the end of a 32768-token prompt
        dict(choose, name="choose for a chunk", seqs=1, longs=1, chunk=4096, context=28672, hq=28, hk=4, keep=51,
             shape=11),
        # long documents: four chunks over 131072 tokens, with a floor under the scores
        dict(choose, name="choose for long chunks", seqs=4, longs=4, chunk=8192, context=122880, hq=28, hk=4, keep=205,
             floor=True, shape=12),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    hq, hk = rng.choice([(32, 8), (28, 4), (8, 8), (8, 2), (16, 2), (12, 4), (4, 4)])
    case = dict(op=rng.choice(["attend", "append", "choose"]), hq=hq, hk=hk, shape=rng.randrange(1 << 20))
    case["seqs"] = spread(1, 48)
    case["longs"] = rng.choice([0, 1, min(2, case["seqs"]), case["seqs"]])
    case["context"] = spread(1, 24000)
    most = {"attend": 2048, "append": 8192, "choose": 8192}[case["op"]]
    case["chunk"] = spread(1, max(1, most // max(1, case["longs"])))
    # the sum of all contexts stays within what a pool of a few hundred MB holds
    case["context"] = max(1, min(case["context"], 65536 // case["seqs"]))
    if case["op"] == "choose":
        case.update(keep=spread(1, 256), floor=rng.random() < 0.3)
        return case
    case.update(dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
                dtype=rng.choice(["bf16", "bf16", "f16"]))
    if case["op"] == "attend":
        case.update(keep=rng.choice([0, 0, spread(1, 64), spread(1, 64)]), per_head=rng.random() < 0.3)
    else:
        case.update(rot=rng.choice([case["dim"], case["dim"] // 2, case["dim"] // 4]), mixed=rng.random() < 0.4,
                    scaling=rng.choice(["none", "linear", "yarn", "llama3"]), base=rng.choice([10000.0, 500000.0]))
        case["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
    return case


def lengths(case):
    """(new tokens, tokens before them) of each sequence: ``longs`` sequences bring chunks, the others one
    token; contexts lie between a third of ``context`` and all of it. Fixed by the case."""
    rng = random.Random(case["shape"])
    new = [case["chunk"] if b < case["longs"] else 1 for b in range(case["seqs"])]
    if case["longs"] > 1:  # chunks of a step differ
        new = [n if b == 0 or n == 1 else max(1, n - rng.randrange(0, 1 + n // 8)) for b, n in enumerate(new)]
    before = [case["context"] if case["seqs"] == 1 else rng.randint(case["context"] // 3, case["context"])
              for _ in new]
    return new, before


def grid(case):
    """(rows of q-blocks in the lists, k-blocks in a row)."""
    new, before = lengths(case)
    return (max(new) + 126) // BLOCK, max((n + c + BLOCK - 1) // BLOCK for n, c in zip(new, before))


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + case["shape"])
    new, before = lengths(case)
    total, nb = [n + c for n, c in zip(new, before)], grid(case)
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    s = dict(case=case, new=new, before=before, cu=cu, nb=nb, max_new=max(new),
             kv_len=torch.tensor(total, dtype=torch.int32, device=DEV))
    hq, hk = case["hq"], case["hk"]
    if case["op"] == "choose":
        # gate scores lie close around a half: sigmoid of small logits, fp32
        s["scores"] = torch.sigmoid(0.02 * torch.randn(len(new), hq, *nb, device=DEV, generator=g))
        s["tau"] = 257 / 512 if case["floor"] else None
        return s
    dt, dim, page = DTYPES[case["dtype"]], case["dim"], case["page"]
    pages = [(t + page - 1) // page for t in total]
    # a pool whose pages are handed out in no order; unused table entries are -1
    perm = torch.randperm(sum(pages) + 3, device=DEV, generator=g, dtype=torch.int32)
    first = torch.tensor([sum(pages[:b]) for b in range(len(pages))], device=DEV)
    at = torch.arange(max(pages), device=DEV).view(1, -1)
    used = at < torch.tensor(pages, device=DEV).view(-1, 1)
    s["table"] = torch.where(used, perm[(first.view(-1, 1) + at).clamp(max=perm.numel() - 1)], -1).to(torch.int32)
    shape = (perm.numel(), page, hk, dim)
    s["k_pages"] = torch.randn(shape, device=DEV, generator=g).to(dt)
    s["v_pages"] = torch.randn(shape, device=DEV, generator=g).to(dt)
    if case["op"] == "attend":
        s["q"] = torch.randn(sum(new), hq, dim, device=DEV, generator=g).to(dt)
        s["idx"] = s["cnt"] = None
        if case["keep"]:
            s["idx"], s["cnt"] = some_lists(case, s, g)
        return s
    # the rows of a fused projection: q, k and v of a token beside one another
    rows = torch.randn(sum(new), hq + 2 * hk, dim, device=DEV, generator=g).to(dt)
    s["q"], s["k"], s["v"] = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
    freq, s["factor"] = frequencies(case)
    s["inv_freq"] = torch.tensor(freq, dtype=torch.float64, device=DEV)
    s["pooled_k"] = torch.zeros(len(new), hk, nb[1], dim, device=DEV)
    return s


def some_lists(case, s, g):
    """Kept lists as the gate gives them: the first block, the q-block's own and others by score."""
    heads = case["hq"] if case["per_head"] else case["hk"]
    nbq, nbk = s["nb"]
    j = torch.arange(nbk, device=DEV)
    row = torch.arange(nbq, device=DEV).view(1, 1, -1, 1)
    ctx = torch.tensor(s["before"], device=DEV).view(-1, 1, 1, 1)
    last = (s["kv_len"].view(-1, 1, 1, 1) - 1) // BLOCK
    own_block = ctx // BLOCK + row
    r = torch.rand(len(s["new"]), heads, nbq, nbk, device=DEV, generator=g)
    r = r + 4.0 * (j == own_block) + 2.0 * (j == 0)
    r = torch.where((j <= own_block) & (own_block <= last), r, -1.0)
    top = torch.topk(r, min(case["keep"], nbk), dim=-1)
    idx = torch.where(top.values >= 0, top.indices, nbk).sort(dim=-1).values
    cnt = (idx < nbk).sum(-1)
    return torch.where(idx < nbk, idx, -1).to(torch.int32).contiguous(), cnt.to(torch.int32).contiguous()


def frequencies(case):
    """Rotary frequencies (radians per position) of the rotated part, and the factor on cos and sin."""
    half, base = case["rot"] // 2, case["base"]
    f = [base ** (-2.0 * i / case["rot"]) for i in range(half)]
    if case["scaling"] == "linear":
        return [x / 4.0 for x in f], 1.0
    if case["scaling"] == "llama3":  # long wavelengths are stretched eightfold, short ones kept, a blend between
        turns = [8192 * x / (2 * math.pi) for x in f]
        blend = [min(1.0, max(0.0, (t - 1.0) / (4.0 - 1.0))) for t in turns]
        return [x * (b + (1 - b) / 8.0) for x, b in zip(f, blend)], 1.0
    if case["scaling"] == "yarn":  # fourfold, by the number of turns within 32768 positions
        lo, hi = (case["rot"] * math.log(32768 / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), case["rot"] - 1)
        ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3))) for i in range(half)]
        return [x * ((1 - r) + r / 4.0) for x, r in zip(f, ramp)], 0.1 * math.log(4.0) + 1.0
    return f, 1.0


# ----------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"attend": own_attend, "append": own_append, "choose": own_choose}[op](s)
    return {"attend": plain_attend, "append": plain_append, "choose": plain_choose}[op](s)


def own_attend(s):
    import tasft_b200 as T

    kept = None if s["idx"] is None else T.KeptBlocks(s["idx"], s["cnt"])
    return T.bsa_chunk_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_len"], s["max_new"], kept,
                             BLOCK)


def own_append(s):
    import tasft_b200 as T

    q, pooled_q = T.rope_append_paged(s["q"], s["k"], s["v"], s["inv_freq"], s["k_pages"], s["v_pages"], s["table"],
                                      s["cu"], s["kv_len"], s["max_new"], interleaved=s["case"]["mixed"],
                                      attention_scaling=s["factor"], pooled_k=s["pooled_k"], block=BLOCK)
    return [q, pooled_q, s["pooled_k"], s["k_pages"], s["v_pages"]]


def own_choose(s):
    import tasft_b200 as T

    kept = T.select_blocks(s["scores"], s["case"]["hk"], s["cu"], s["kv_len"], s["case"]["keep"], tau=s["tau"],
                           block=BLOCK)
    return [kept.idx, kept.cnt]


def plain_attend(s):
    """softmax(q k^T / sqrt(D)) v over the kept keys up to each token's own position, in fp32.
    Sequences with as many new tokens as one another are computed together."""
    case, new, before = s["case"], s["new"], s["before"]
    hq, hk, dim, page = case["hq"], case["hk"], case["dim"], case["page"]
    out = torch.empty_like(s["q"])
    for n in sorted(set(new)):
        which = [b for b, m in enumerate(new) if m == n]
        b = torch.tensor(which, device=DEV)
        longest = max(before[x] for x in which) + n
        rows = s["cu"][b].long().view(-1, 1) + torch.arange(n, device=DEV)
        q = s["q"][rows].float().view(len(which), n, hk, hq // hk, dim)
        t = s["table"][b, :(longest + page - 1) // page].long().clamp(min=0)
        k = s["k_pages"][t].flatten(1, 2)[:, :longest].float()
        v = s["v_pages"][t].flatten(1, 2)[:, :longest].float()
        scores = torch.einsum("bnhgd,blhd->bhgnl", q, k) * (1.0 / math.sqrt(dim))
        j = torch.arange(longest, device=DEV)
        pos = (s["kv_len"][b] - n).view(-1, 1) + torch.arange(n, device=DEV)
        seen = (j <= pos.unsqueeze(-1)).view(len(which), 1, 1, n, longest)
        if s["idx"] is not None:
            row = pos // BLOCK - ((s["kv_len"][b] - n) // BLOCK).view(-1, 1)
            idx = s["idx"][b].long()
            keep = torch.zeros(*idx.shape[:3], s["nb"][1] + 1, dtype=torch.bool, device=DEV)
            keep = keep.scatter_(-1, torch.where(idx < 0, s["nb"][1], idx), True)
            keep = keep.gather(2, row.view(len(which), 1, n, 1).expand(-1, idx.shape[1], -1, keep.shape[-1]))
            keep = keep[..., j // BLOCK]
            seen = seen & keep.view(len(which), hk, -1, n, longest)
        scores = scores.masked_fill_(~seen, -math.inf)
        top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
        p = scores.sub_(top).exp_()
        norm = p.sum(-1, keepdim=True)
        o = torch.einsum("bhgnl,blhd->bnhgd", p.div_(torch.where(norm > 0, norm, 1.0)), v)
        out[rows] = o.reshape(len(which), n, hq, dim).to(out.dtype)
    return out


def token_rows(s):
    """(sequence, position) of each new token, and its row in the page pools."""
    b = torch.repeat_interleave(torch.arange(len(s["new"]), device=DEV), torch.diff(s["cu"]).long(),
                                output_size=s["q"].shape[0])
    pos = (s["kv_len"] - s["cu"][1:]).long()[b] + torch.arange(s["q"].shape[0], device=DEV)
    page = s["case"]["page"]
    return b, pos, s["table"][b, pos // page].long() * page + pos % page


def rotate(x, cos, sin, case):
    """fp32 rotation of the first ``rot`` columns: pairs (i, i + rot/2), or (2i, 2i+1) when mixed."""
    rot = case["rot"]
    x = x.float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if case["mixed"] else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((c, d), -1).flatten(-2) if case["mixed"] else torch.cat((c, d), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def plain_append(s):
    case, hk, dim = s["case"], s["case"]["hk"], s["case"]["dim"]
    b, pos, slot = token_rows(s)
    angle = pos.double().unsqueeze(-1) * s["inv_freq"]
    cos, sin = ((f(angle) * s["factor"]).float().unsqueeze(1) for f in (torch.cos, torch.sin))
    q = rotate(s["q"], cos, sin, case).to(s["q"].dtype)
    k = rotate(s["k"], cos, sin, case).to(s["k"].dtype)
    flat_k, flat_v = s["k_pages"].view(-1, hk, dim), s["v_pages"].view(-1, hk, dim)
    flat_k[slot] = k
    flat_v[slot] = s["v"]
    # block means of the rows that are there (the rest of a block counts as zeros): of the new
    # queries, and of the cached keys of every block that got new ones
    nbq, page = s["nb"][0], case["page"]
    start = (s["kv_len"] - torch.diff(s["cu"])).long()
    lo = start // BLOCK * BLOCK
    at = lo.view(-1, 1) + torch.arange(nbq * BLOCK, device=DEV)
    there = (at < s["kv_len"].view(-1, 1)).view(len(s["new"]), -1, 1, 1)
    fresh = there & (at >= start.view(-1, 1)).view(len(s["new"]), -1, 1, 1)
    row = (s["cu"][:-1].view(-1, 1) + at - start.view(-1, 1)).clamp(0, q.shape[0] - 1)
    pooled_q = torch.where(fresh, q[row].float(), 0.0).unflatten(1, (nbq, BLOCK)).sum(2) / BLOCK
    cached = s["table"].gather(1, (at // page).clamp(max=s["table"].shape[1] - 1)).long().clamp(min=0) * page + at % page
    means = torch.where(there, flat_k[cached].float(), 0.0).unflatten(1, (nbq, BLOCK)).sum(2) / BLOCK
    touched = (at[:, ::BLOCK] < s["kv_len"].view(-1, 1)).nonzero(as_tuple=True)
    s["pooled_k"][touched[0], :, lo[touched[0]] // BLOCK + touched[1]] = means[touched]
    return [q, pooled_q.transpose(1, 2).contiguous(), s["pooled_k"], s["k_pages"], s["v_pages"]]


def plain_choose(s):
    """Per KV head and row: the first block, the row's own and the best of the others, ``keep`` in
    all; a block's score is the highest of the group's heads, ties go to the lowest index."""
    case, (nbq, nbk) = s["case"], s["nb"]
    n, hk = len(s["new"]), case["hk"]
    score = s["scores"].view(n, hk, -1, nbq, nbk).amax(2)
    j = torch.arange(nbk, device=DEV)
    last = ((s["kv_len"] - 1) // BLOCK).view(-1, 1, 1, 1)
    mine = ((s["kv_len"] - torch.diff(s["cu"])) // BLOCK).view(-1, 1, 1, 1) + torch.arange(nbq, device=DEV).view(-1, 1)
    forced = ((j == 0) | (j == mine)) & (j <= mine) & (mine <= last)
    other = (j > 0) & (j < mine) & (mine <= last)
    if s["tau"] is not None:
        other = other & (score >= s["tau"])
    order = torch.where(other, score, -math.inf).sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, j.expand_as(order))
    kept = forced | (other & (rank < case["keep"] - forced.sum(-1, keepdim=True)))
    width = min(nbk, max(case["keep"], 2))
    idx = torch.where(kept, j, nbk).sort(dim=-1).values[..., :width]
    return [torch.where(idx < nbk, idx, -1).to(torch.int32), kept.sum(-1).to(torch.int32)]


# ----------------------------------------------------------------------------- what a pass needs
def work(case):
    new, before = lengths(case)
    nbq, nbk = grid(case)
    hq, hk, tokens = case["hq"], case["hk"], sum(new)
    if case["op"] == "choose":
        # the scores up to each row's own block; lists and counts
        rows = [(c // BLOCK + i) for n, c in zip(new, before) for i in range((c + n - 1) // BLOCK - c // BLOCK + 1)]
        read = sum(r + 1 for r in rows) * hq * 4
        width = min(nbk, max(case["keep"], 2))
        return {"bytes": read + len(new) * hk * nbq * (width + 1) * 4, "flops": sum(r + 1 for r in rows) * hq}
    size, dim = DTYPES[case["dtype"]].itemsize, case["dim"]
    if case["op"] == "append":
        moved = 2 * tokens * (hq + 2 * hk) * dim * size
        blocks = sum((c + n - 1) // BLOCK - c // BLOCK + 1 for n, c in zip(new, before))
        old = sum(c % BLOCK for c in before) * hk * dim * size  # keys of the blocks begun earlier
        means = len(new) * hq * nbq * dim * 4 + blocks * hk * dim * 4
        return {"bytes": moved + old + means, "flops": tokens * (hq + hk) * (case["rot"] * 3 + dim)}
    heads = hq if case["per_head"] else hk
    pairs = keys = lists = 0
    for n, c in zip(new, before):
        first, last = c // BLOCK, (c + n - 1) // BLOCK
        left = 1.0  # the share of earlier blocks that no row has kept
        for own_block in range(first, last + 1):
            lo, hi = max(c, own_block * BLOCK), min(c + n, (own_block + 1) * BLOCK)
            full = own_block if not case["keep"] else min(case["keep"] - 1, own_block)
            pairs += (hi - lo) * full * BLOCK + sum(p - own_block * BLOCK + 1 for p in range(lo, hi))
            left *= 1.0 - full / max(1, own_block)
            lists += (full + 2) * 4
        if case["per_head"] and case["keep"]:
            left = left ** (hq // hk)
        keys += first * BLOCK * (1.0 - left) + (c + n - first * BLOCK)
    kept = lists * heads if case["keep"] else 0
    return {"bytes": int(2 * tokens * hq * dim * size + 2 * keys * hk * dim * size + kept),
            "flops": int(4 * pairs * hq * dim)}


# ----------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": exact_attend, "append": exact_append, "choose": exact_choose}[case["op"]](s)


def exact_attend(s):
    """Token position by position of the definition: one sequence and one KV head at a time."""
    case = s["case"]
    page, hq, hk = case["page"], case["hq"], case["hk"]
    group = hq // hk
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    start = 0
    for b, (n, c) in enumerate(zip(s["new"], s["before"])):
        keys = torch.arange(n + c, device=DEV)
        pool = s["table"][b].long()[keys // page], keys % page
        place = c + torch.arange(n, device=DEV)
        for h in range(hk):
            k, v = s["k_pages"][pool[0], pool[1], h].double(), s["v_pages"][pool[0], pool[1], h].double()
            for u in range(h * group, (h + 1) * group):
                e = (s["q"][start:start + n, u].double() @ k.T) / math.sqrt(case["dim"])
                mask = keys.view(1, -1) > place.view(-1, 1)
                if s["idx"] is not None:
                    lists = s["idx"][b, u if case["per_head"] else h].long()
                    at = (lists.unsqueeze(-1) == torch.arange(s["nb"][1], device=DEV)).any(1)
                    mask |= ~at[place // BLOCK - c // BLOCK][:, keys // BLOCK]
                e[mask] = -math.inf
                p = torch.exp(e - e.max(dim=1, keepdim=True).values.clamp(min=-1e300))
                total = p.sum(1, keepdim=True)
                out[start:start + n, u] = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
        start += n
    return out


def exact_append(s):
    """Complex turns: a pair (x, y) is x + iy, times exp(i * angle) * factor. The block means are of
    values as they are held, rounded to the tensors' type, and have no value of their own in 64 bits."""
    case, page, rot = s["case"], s["case"]["page"], s["case"]["rot"]
    kp, vp, q_out = s["k_pages"].double(), s["v_pages"].double(), s["q"].double()
    even, odd = torch.arange(0, rot, 2), torch.arange(1, rot, 2)
    if not case["mixed"]:
        even, odd = torch.arange(rot // 2), torch.arange(rot // 2) + rot // 2
    start = 0
    for b, (n, c) in enumerate(zip(s["new"], s["before"])):
        place = c + torch.arange(n, device=DEV)
        turn = torch.polar(torch.full((n, rot // 2), s["factor"], dtype=torch.float64, device=DEV),
                           place.view(-1, 1).double() * s["inv_freq"]).unsqueeze(1)
        rows, table = slice(start, start + n), s["table"][b].long()
        turned = []
        for x in (s["q"][rows].double(), s["k"][rows].double()):
            z = torch.complex(x[..., even], x[..., odd]) * turn
            x[..., even], x[..., odd] = z.real, z.imag
            turned.append(x)
        q_out[rows] = turned[0]
        kp[table[place // page], place % page] = turned[1]
        vp[table[place // page], place % page] = s["v"][rows].double()
        start += n
    return [q_out, None, None, kp, vp]


def exact_choose(s):
    """A block's rank is the number of blocks that beat it; written over rows of one sequence."""
    case, (nbq, nbk) = s["case"], s["nb"]
    hk, group = case["hk"], case["hq"] // case["hk"]
    width = min(nbk, max(case["keep"], 2))
    idx = torch.full((len(s["new"]), hk, nbq, width), -1, dtype=torch.int32)
    cnt = torch.zeros(len(s["new"]), hk, nbq, dtype=torch.int32)
    for b, (n, c) in enumerate(zip(s["new"], s["before"])):
        for i in range((c + n - 1) // BLOCK - c // BLOCK + 1):
            mine = c // BLOCK + i
            best = s["scores"][b, :, i, :mine + 1].double().unflatten(0, (hk, group)).max(dim=1).values
            a, z = best.unsqueeze(-1), best.unsqueeze(-2)
            j = torch.arange(mine + 1, device=DEV)
            free = (j > 0) & (j < mine)
            ok = free & (best >= s["tau"]) if s["tau"] is not None else free.expand_as(best)
            beats = ((z > a) | ((z == a) & (j.view(1, -1) < j.view(-1, 1)))) & ok.unsqueeze(-2)
            take = ok & (beats.sum(-1) < case["keep"] - (1 if mine == 0 else 2))
            take = (take | ~free).cpu()
            for h in range(hk):
                got = take[h].nonzero().flatten().to(torch.int32)
                idx[b, h, i, :len(got)] = got
                cnt[b, h, i] = len(got)
    return [idx, cnt]
