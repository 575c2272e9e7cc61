"""The path of a token through a layer with the paged 4-bit cache: pages and places, fused q/k/v, rotary embedding, store, attention,
output projection - prompts, single tokens, requests that arrive and end, eager and as a captured step."""
import numpy as np
import pytest
import torch

from tests.attention_reference import as_held, attention, bound
from tests.test_gpu_decoder_layer import HEAD_DIM, HEADS, HIDDEN, KV_HEADS, PRUNED_DIM, make_layers
from tests.test_oracle_fused_rope import rope_tables

pytestmark = pytest.mark.gpu
ROWS, PAGE, MOST = 4, 16, 64


class Layer:
    def __init__(self, dev):
        from uniql_amd.quantize.fused_layers import W4A16FusedLinear
        from uniql_amd.quantize.quant_kv_cache import KVPages, W4KVCache
        L = make_layers(dev, True)
        self.qkv, self.o = W4A16FusedLinear.from_linears([L["q"], L["k"], L["v"]]), L["o"]
        cos, sin, _ = rope_tables(MOST * 4, HEAD_DIM)
        self.cos, self.sin = torch.from_numpy(cos).to(dev).view(-1, HEAD_DIM), torch.from_numpy(sin).to(dev).view(-1, HEAD_DIM)
        first = np.sort(np.random.default_rng(0).choice(HEAD_DIM // 2, PRUNED_DIM // 2, replace=False))
        self.idx = torch.from_numpy(np.tile(np.concatenate((first, first + HEAD_DIM // 2)), (KV_HEADS, 1))).to(torch.uint8).to(dev)
        self.pages = KVPages(12, PAGE, ROWS, 5, device=dev)
        self.cache = W4KVCache(12, PAGE, KV_HEADS, PRUNED_DIM, device=dev)
        self.dev = dev

    def project(self, x, step):
        from uniql_amd import ops
        q, k, v = self.qkv(x)
        n = x.shape[0]
        q, k, v = q.reshape(1, n, HEADS, PRUNED_DIM), k.reshape(1, n, KV_HEADS, PRUNED_DIM), v.reshape(n, KV_HEADS, PRUNED_DIM)
        q, k = q.contiguous(), k.contiguous()
        ops.rope_indices_(q, k, self.cos[step.positions][None], self.sin[step.positions][None], self.idx)
        return q[0], k[0], v

    def step(self, x, new, out):
        step = self.pages.assign(new, x.shape[0])
        q, k, v = self.project(x, step)
        self.cache.store(k, v, step.slots)
        a = self.cache.attend(q, self.pages.table, self.pages.lengths, cu_q=step.cu, out=out)
        return step, q, k, v, a, self.o(a.view(x.shape[0], -1))


def test_prompts_then_tokens(gpu):
    from uniql_amd.attention import prompt_attention
    layer = Layer(gpu)
    gen = torch.Generator().manual_seed(4)
    history = [[torch.empty(0, KV_HEADS, PRUNED_DIM).half()] * 2 for _ in range(ROWS)]
    scale = PRUNED_DIM ** -0.5
    for number, new in enumerate([[5, 0, 17, 1], [1, 0, 1, 1], [1, 20, -1, 1], [1, 1, 30, 0], [2, 1, 1, 1], [1, 1, 90, 1], [-1, 1, 1, 40]]):
        tokens = sum(max(n, 0) for n in new)
        x = (torch.randn(tokens + 3, HIDDEN, generator=gen) * 0.5).half().to(gpu)   # three padding rows
        out = torch.full((tokens + 3, HEADS, PRUNED_DIM), 9.0, device=gpu).half()
        step, q, k, v, a, y = layer.step(x, torch.tensor(new, dtype=torch.int32, device=gpu), out)
        assert y.shape == x.shape
        refused = step.refused.tolist()
        assert refused == [0, 0, 0, 0] if number < 5 else True
        if number == 5:
            assert refused == [0, 0, 1, 0]      # 90 tokens do not fit a row of five pages
        assert (a[tokens:] == 9).all() and (step.slots[tokens:] == -1).all()
        prompt = prompt_attention(q, k, v, step.cu) if number == 0 else None
        cu = step.cu.tolist()
        for r, n in enumerate(new):
            if n < 0:
                history[r] = [torch.empty(0, KV_HEADS, PRUNED_DIM).half()] * 2
            if n <= 0 or refused[r]:
                continue
            rows = slice(cu[r], cu[r + 1])
            history[r] = [torch.cat((h, t[rows].cpu())) for h, t in zip(history[r], (k, v))]
            held_k, (held_v, v_scale) = as_held(history[r][0])[0], as_held(history[r][1])
            seen = history[r][0].shape[0]
            assert step.positions[rows].tolist() == list(range(seen - n, seen))
            o, mean_abs, spread = attention(q[rows].cpu(), held_k, held_v, scale, seen - n + 1)
            held = attention(q[rows].cpu(), held_k, v_scale.unsqueeze(-1), scale, seen - n + 1)[0]
            assert ((a[rows].cpu().double() - o).abs() <= bound(o, mean_abs, spread, seen, held)).all()
            if prompt is not None:
                p = attention(q[rows].cpu(), history[r][0], history[r][1], scale, 1)
                assert ((prompt[rows].cpu().double() - p[0]).abs() <= bound(*p, seen)).all()
        assert layer.pages.lengths.tolist() == [h[0].shape[0] for h in history]


def test_a_prompt_in_pieces_reads_the_cache(gpu):
    """a piece's queries over the earlier pieces from the cache and its own keys, all read back as fp16: the same as over the cache"""
    from uniql_amd.attention import prompt_attention
    layer = Layer(gpu)
    gen = torch.Generator().manual_seed(8)
    for new in ([20, 3, 0, 7], [11, 16, 5, 1]):
        tokens = sum(new)
        x = (torch.randn(tokens, HIDDEN, generator=gen) * 0.5).half().to(gpu)
        step, q, k, v, a, _ = layer.step(x, torch.tensor(new, dtype=torch.int32, device=gpu), None)
        lengths = layer.pages.lengths
        cu_k = torch.cat((torch.zeros(1, dtype=torch.int32, device=gpu), torch.cumsum(lengths, 0).int()))
        held_k, held_v = layer.cache.load(layer.pages.table, cu_k, int(cu_k[-1]))
        b = prompt_attention(q, held_k, held_v, step.cu, cu_k)
        # the values read back are rounded to fp16 once more (half a step, 2^-11), keys too, which moves scores of about ten by 2^-8
        assert (a.float() - b.float()).abs().max() <= 2 ** -6 * a.float().abs().max()


def test_a_captured_step_replayed(gpu):
    """assign, store and attend in one graph: lengths grow from replay to replay as they do eagerly"""
    layer, eager = Layer(gpu), Layer(gpu)
    gen = torch.Generator().manual_seed(6)
    x = (torch.randn(32, HIDDEN, generator=gen) * 0.5).half().to(gpu)
    new = torch.tensor([9, 0, 12, 11], dtype=torch.int32, device=gpu)
    for l in (layer, eager):
        l.step(x, new, None)
    x = x[:ROWS].clone()
    new = torch.tensor([1, 1, 1, 1], dtype=torch.int32, device=gpu)
    state = [b.clone() for m in (layer.pages, layer.cache) for b in m.buffers()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer.step(x, new, None)
    stream.synchronize()
    for b, old in zip([b for m in (layer.pages, layer.cache) for b in m.buffers()], state):
        b.copy_(old)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = layer.step(x, new, None)
    for i in range(7):
        x.copy_((torch.randn(ROWS, HIDDEN, generator=gen) * 0.5).half())
        if i == 4:
            new.copy_(torch.tensor([1, -1, 1, 1], dtype=torch.int32))
        if i == 5:
            new.fill_(1)
        torch.cuda.synchronize()
        graph.replay()
        want = eager.step(x, new, None)
        torch.cuda.synchronize()
        n = int(new.clamp_min(0).sum())
        for got, w in zip(captured[0][:1] + captured[0][2:] + captured[1:], want[0][:1] + want[0][2:] + want[1:]):
            assert torch.equal(got[:n] if got.shape[0] == ROWS and i == 4 else got, w[:n] if w.shape[0] == ROWS and i == 4 else w)
        assert layer.pages.lengths.tolist() == eager.pages.lengths.tolist()
        assert torch.equal(layer.pages.table, eager.pages.table)
