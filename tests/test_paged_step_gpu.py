"""A serving step as it is used: rotary append, gate from the block means, choice of blocks,
attention over the cache, chunk after chunk; captured, and on two streams at once."""
from __future__ import annotations

import math

import pytest
import torch

import paged_oracle as R
import tasft_b200 as T

pytestmark = pytest.mark.gpu
DEV = "cuda"
HQ, HK, D, PAGE, NBK = 8, 2, 128, 16, 20
SCALING = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096)


class Layer:
    """One layer's cache for B sequences, its gate, and the step over them."""

    def __init__(self, B, seed=0, top_k=5):
        g = torch.Generator(device=DEV).manual_seed(seed)
        per = NBK * 64 // PAGE
        self.kp = torch.full((B * per + 2, PAGE, HK, D), float("nan"), device=DEV, dtype=torch.bfloat16)
        self.vp = self.kp.clone()
        self.table = torch.randperm(B * per, generator=g, device=DEV).to(torch.int32).view(B, per)
        self.means = torch.zeros(B, HK, NBK, D, device=DEV)
        self.freq, self.factor = T.rope_inv_freq(D, 500000.0, SCALING, device=DEV)
        torch.manual_seed(seed)
        # rows are chunk rows, not blocks: the choice below applies the causal order
        self.gate = T.AttnGate(HQ, D, block_size=64, is_causal=False).to(DEV)
        torch.nn.init.normal_(self.gate.gate_proj_out.weight, std=1.0)
        self.top_k = top_k

    def step(self, rows, cu, kv_len, max_new):
        q, k, v = rows[:, :HQ], rows[:, HQ:HQ + HK], rows[:, HQ + HK:]
        self.q, self.pooled_q = T.rope_append_paged(q, k, v, self.freq, self.kp, self.vp, self.table, cu, kv_len, max_new,
                                                    attention_scaling=self.factor, pooled_k=self.means)
        n = self.pooled_q.shape[2]
        with torch.no_grad():
            self.soft = self.gate.forward_pooled(self.pooled_q, self.means, n * 64, NBK * 64).soft_scores
        self.kept = T.select_blocks(self.soft, HK, cu, kv_len, self.top_k)
        return T.bsa_chunk_paged(self.q, self.kp, self.vp, self.table, cu, kv_len, max_new, self.kept)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cu_of(new):
    return ints([sum(new[:b]) for b in range(len(new) + 1)])


def check_step(layer, out, new, ctx):
    idx, cnt = R.choose(layer.soft, HK, new, ctx, layer.top_k)
    assert torch.equal(layer.kept.idx.cpu(), idx) and torch.equal(layer.kept.cnt.cpu(), cnt)
    o, a = R.attend(layer.q, layer.kp, layer.vp, layer.table, new, ctx, (layer.kept.idx, layer.kept.cnt))
    bound = R.attend_bound(o, a, torch.bfloat16, max(n + c for n, c in zip(new, ctx)))
    assert ((out.double() - o).abs() <= bound).all()


def test_prompts_in_chunks_then_tokens():
    layer = Layer(3)
    g = torch.Generator(device=DEV).manual_seed(1)
    ctx = [0, 0, 0]
    prompts = [[], [], []]
    for new in ([200, 63, 1], [100, 500, 1], [1, 1, 300], [1, 0, 1], [1, 1, 1]):
        rows = torch.randn(sum(new), HQ + 2 * HK, D, generator=g, device=DEV).to(torch.bfloat16)
        out = layer.step(rows, cu_of(new), ints([n + c for n, c in zip(new, ctx)]), max(new))
        check_step(layer, out, new, ctx)
        at = 0
        for b, n in enumerate(new):
            prompts[b].append(rows[at:at + n])
            at += n
        ctx = [n + c for n, c in zip(new, ctx)]
    # the means kept along the way are those of the rotated keys as a whole
    for b in range(3):
        x = torch.cat(prompts[b])
        want = R.rotate(x[:, HQ:HQ + HK], torch.arange(ctx[b], device=DEV), layer.freq, layer.factor, False)
        held = R.cached(layer.kp, layer.table[b], ctx[b]).double()
        assert ((held - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18).all()
        for blk in range((ctx[b] + 63) // 64):
            mean = held[blk * 64:(blk + 1) * 64].sum(0) / 64
            assert ((layer.means[b, :, blk] - mean).abs() <= 65 * 2.0 ** -24 * held.abs().amax()).all()


def test_a_captured_step_replays_on_new_lengths():
    layer = Layer(2, seed=3)
    rows = torch.randn(70, HQ + 2 * HK, D, device=DEV).to(torch.bfloat16)
    cu, kv_len = cu_of([64, 6]), ints([64, 6])
    out = torch.empty(70, HQ, D, device=DEV, dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(rows, cu, kv_len, 64)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out.copy_(layer.step(rows, cu, kv_len, 64))
    ctx = [0, 0]
    for new in ([64, 6], [10, 60], [1, 1], [0, 64]):
        rows.copy_(torch.randn(70, HQ + 2 * HK, D, device=DEV))
        cu.copy_(cu_of(new))
        kv_len.copy_(ints([n + c for n, c in zip(new, ctx)]))
        graph.replay()
        torch.cuda.synchronize()
        n = sum(new)
        q, o = layer.q, out
        layer.q, part = q[:n], o[:n]
        check_step(layer, part, new, ctx)
        layer.q = q
        ctx = [n + c for n, c in zip(new, ctx)]


def test_two_streams_at_once():
    """Calls on two streams, neither the default one, share nothing."""
    layers = [Layer(2, seed=5), Layer(2, seed=6)]
    streams = [torch.cuda.Stream() for _ in layers]
    new = [[400, 1], [1, 700]]
    rows = [torch.randn(sum(n), HQ + 2 * HK, D, device=DEV).to(torch.bfloat16) for n in new]
    args = [(cu_of(n), ints(n), max(n)) for n in new]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                outs[i].append(layers[i].step(rows[i], *args[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        check_step(layers[i], outs[i][0], new[i], [0, 0])
        for o in outs[i][1:]:
            assert torch.equal(o, outs[i][0])


def test_decode_takes_the_chosen_lists():
    layer = Layer(2, seed=8)
    rows = torch.randn(900, HQ + 2 * HK, D, device=DEV).to(torch.bfloat16)
    layer.step(rows, cu_of([300, 600]), ints([300, 600]), 600)
    rows = torch.randn(2, HQ + 2 * HK, D, device=DEV).to(torch.bfloat16)
    kv_len = ints([301, 601])
    out = layer.step(rows, cu_of([1, 1]), kv_len, 1)
    # the older call multiplies 0 by what the cache holds behind the last token: zeros there
    layer.kp.nan_to_num_(0.0)
    layer.vp.nan_to_num_(0.0)
    one = T.bsa_decode_paged(layer.q, layer.kp, layer.vp, layer.table, kv_len,
                             T.KeptBlocks(layer.kept.idx[:, :, 0], layer.kept.cnt[:, :, 0]))
    o, a = R.attend(layer.q, layer.kp, layer.vp, layer.table, [1, 1], [300, 600], (layer.kept.idx, layer.kept.cnt))
    bound = R.attend_bound(o, a, torch.bfloat16, 601)
    assert ((out.double() - o).abs() <= bound).all() and ((one.double() - o).abs() <= bound).all()
    assert math.isfinite(float(one.float().abs().max()))
