"""Plain 64-bit restatements of the paged serving operators, and batches to run them on."""
from __future__ import annotations

import math

import torch

BLK = 64


def layout(new, ctx, page, Hk, D, dtype, dev, gen, spare=3, fill=None):
    """Page pools in shuffled order for sequences of ``ctx + new`` tokens; rows that no token owns
    hold ``fill`` (random values when None). Returns k_pages, v_pages, table, cu, kv_len."""
    total = [n + c for n, c in zip(new, ctx)]
    need = [(t + page - 1) // page for t in total]
    P = sum(need) + spare
    perm = torch.randperm(P, generator=gen, device=dev)
    kp = torch.randn(P, page, Hk, D, generator=gen, device=dev).to(dtype)
    vp = torch.randn(P, page, Hk, D, generator=gen, device=dev).to(dtype)
    table = torch.full((len(new), max(max(need), 1)), -1, dtype=torch.int32, device=dev)
    owned = torch.zeros(P, page, dtype=torch.bool, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n].to(torch.int32)
        at += n
        t = torch.arange(total[b], device=dev)
        owned[table[b].long()[t // page], t % page] = True
    if fill is not None:
        kp[~owned] = fill
        vp[~owned] = fill
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=dev)
    return kp, vp, table, cu, torch.tensor(total, dtype=torch.int32, device=dev)


def cached(pool, table_row, n):
    """The first n rows of a sequence, [n, Hk, D]."""
    page = pool.shape[1]
    t = torch.arange(n, device=pool.device)
    return pool[table_row.long()[t // page], t % page]


def random_lists(new, ctx, heads, width, dev, gen, density=0.4, own=True, empty=0.0):
    """Ascending kept lists [B, heads, rows, width] with -1 padding, and counts."""
    rows = (max(new) + 126) // BLK
    idx = torch.full((len(new), heads, rows, width), -1, dtype=torch.int32)
    cnt = torch.zeros(len(new), heads, rows, dtype=torch.int32)
    cpu = torch.Generator().manual_seed(int(torch.randint(0, 1 << 30, (1,), generator=gen, device=dev).item()))
    for b, (n, c) in enumerate(zip(new, ctx)):
        if n == 0:
            continue
        for h in range(heads):
            for i in range((c + n - 1) // BLK - c // BLK + 1):
                mine = c // BLK + i
                if torch.rand(1, generator=cpu).item() < empty:
                    continue
                keep = torch.rand(mine + 1, generator=cpu) < density
                keep[mine] = own
                got = keep.nonzero().flatten()[-width:]
                idx[b, h, i, :len(got)] = got.to(torch.int32)
                cnt[b, h, i] = len(got)
    return idx.to(dev), cnt.to(dev)


def attend(q, kp, vp, table, new, ctx, kept=None, scale=None):
    """(o, a): the attention output in fp64 and a = sum_j p_j |v_j|, what roundings of p scale with.
    Values behind the mask take no part, whatever they are."""
    T, Hq, D = q.shape
    Hk = kp.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    start = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        if n == 0:
            continue
        k, v = cached(kp, table[b], n + c).double(), cached(vp, table[b], n + c).double()
        pos = c + torch.arange(n, device=q.device)
        j = torch.arange(n + c, device=q.device)
        for h in range(Hq):
            g = h // (Hq // Hk)
            see = j.view(1, -1) <= pos.view(-1, 1)
            if kept is not None:
                idx, cnt = kept
                hm = h if idx.shape[1] == Hq else g
                nb = (n + c + BLK - 1) // BLK
                keep = torch.zeros(idx.shape[2], nb + 1, dtype=torch.bool, device=q.device)
                lists = idx[b, hm].long()
                in_list = torch.arange(lists.shape[1], device=q.device) < cnt[b, hm].view(-1, 1)
                keep.scatter_(1, torch.where(in_list & (lists >= 0) & (lists < nb), lists, nb), True)
                see = see & keep[pos // BLK - c // BLK][:, j // BLK]
            s = (q[start:start + n, h].double() @ k[:, g].T) * scale
            s = torch.where(see, s, -math.inf)
            m = s.amax(1, keepdim=True)
            p = torch.where(see, torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
            norm = p.sum(1, keepdim=True)
            p = p / torch.where(norm == 0, 1.0, norm)
            used = see.any(0)
            vz = torch.where(used.view(-1, 1), v[:, g], 0.0)
            o[start:start + n, h] = p @ vz
            a[start:start + n, h] = p @ vz.abs()
        start += n
    return o, a


def attend_bound(o, a, dtype, keys):
    """How far a kernel that rounds p and o once to ``dtype`` may be off: half a step of o, half a
    step of every p (|sum dp v| <= u a), and 2^-14 a for fp32 scores, exponentials and sums. In
    fp16 a p under 2^-14 is held to 2^-25 absolute, against a sum of at least 1."""
    u = torch.finfo(dtype).eps / 2
    t = u * (o.abs() + a) + 2.0 ** -14 * a + 1e-7
    if dtype == torch.float16:
        t = t + keys * 2.0 ** -25 * 8
    return t


def choose(scores, hk, new, ctx, top_k, tau=None, first=1, local=1, width=None, block=BLK):
    """Kept lists from scores, by sorting (score, lowest index first) row by row."""
    B, Hq, rows, nbk = scores.shape
    width = min(nbk, max(top_k, first + local)) if width is None else width
    idx = torch.full((B, hk, rows, width), -1, dtype=torch.int32)
    cnt = torch.zeros(B, hk, rows, dtype=torch.int32)
    s = scores.double().cpu().view(B, hk, Hq // hk, rows, nbk)
    s = torch.where(torch.isnan(s), -math.inf, s).amax(2)
    for b, (n, c) in enumerate(zip(new, ctx)):
        for i in range((c + n - 1) // block - c // block + 1 if n else 0):
            mine = c // block + i
            forced = sorted(set(range(min(first, mine + 1))) | set(range(max(0, mine + 1 - local), mine + 1)))
            for h in range(hk):
                row = s[b, h, i].tolist()
                free = [j for j in range(mine) if j not in forced and row[j] > -math.inf
                        and (tau is None or row[j] >= tau)]
                free.sort(key=lambda j: (-row[j], j))
                got = sorted(forced + free[:max(0, top_k - len(forced))])
                idx[b, h, i, :len(got)] = torch.tensor(got, dtype=torch.int32)
                cnt[b, h, i] = len(got)
    return idx, cnt


def rotate(x, pos, inv_freq, factor, interleaved):
    """Pairs of the first columns turned by pos * inv_freq, in fp64. x [n, H, D]."""
    x = x.double().clone()
    rot = 2 * inv_freq.numel()
    i = torch.arange(rot // 2, device=x.device)
    e, o = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    ang = pos.double().view(-1, 1, 1) * inv_freq.double().view(1, 1, -1)
    c, s = torch.cos(ang) * factor, torch.sin(ang) * factor
    a, b = x[..., e].clone(), x[..., o].clone()
    x[..., e], x[..., o] = a * c - b * s, b * c + a * s
    return x
