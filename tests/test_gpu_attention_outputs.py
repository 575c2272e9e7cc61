"""Outputs that the caller gives: what shares memory with an input, another output or itself is refused, other ranges of the same
buffer are taken."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_prompt_attention(gpu):
    from uniql_amd.attention import prompt_attention
    n, gen = 40, torch.Generator().manual_seed(1)
    cu = torch.tensor([0, n], dtype=torch.int32, device=gpu)
    fused = torch.randn(n + 1, 4 * 64 + 2 * 64 + 2 * 64 + 4 * 64, generator=gen).half().to(gpu)
    q, k, v, rest = (x[:n].unflatten(1, (-1, 64)) for x in fused.split((256, 128, 128, 256), dim=1))
    before = fused.clone()
    refused = [fused[:n, at:at + 256].unflatten(1, (4, 64)) for at in (1, 200, 255, 256, 300, 500, 511)]
    refused += [fused[1:, 256:512].unflatten(1, (4, 64)), fused[1:, :256].unflatten(1, (4, 64)),
                fused.view(-1)[2000:].as_strided((n, 4, 64), (256, 64, 1))]
    for out in refused:
        with pytest.raises(RuntimeError, match="share memory"):
            prompt_attention(q, k, v, cu, out=out)
    for strides in ((64, 64, 1), (32, 64 * n, 1), (256, 32, 1), (0, 64, 1), (64, 128, 1)):
        with pytest.raises(RuntimeError, match="overlaps itself"):
            prompt_attention(q, k, v, cu, out=torch.zeros(n * 512, device=gpu).half().as_strided((n, 4, 64), strides))
    assert torch.equal(fused, before)
    want = prompt_attention(q, k, v, cu)
    assert prompt_attention(q, k, v, cu, out=rest).data_ptr() == rest.data_ptr()
    assert torch.equal(rest, want) and torch.equal(fused[:, :512], before[:, :512]) and torch.equal(fused[n], before[n])
    turned = torch.zeros(4, n, 64, device=gpu).half().transpose(0, 1)      # head after head
    assert torch.equal(prompt_attention(q, k, v, cu, out=turned), want)
    in_turn = torch.zeros(n, 4, 2, 64, device=gpu).half()                  # heads of q and of the output in turn
    in_turn[:, :, 0] = q
    assert torch.equal(prompt_attention(in_turn[:, :, 0], k, v, cu, out=in_turn[:, :, 1]), want)


def test_attention_over_the_cache_and_loading(gpu):
    from uniql_amd.quantize.quant_kv_cache import W4KVCache
    gen = torch.Generator().manual_seed(2)
    cache = W4KVCache(4, 16, 2, 64, 64, device=gpu)
    x = torch.randn(64, 2, 64, generator=gen).half().to(gpu)
    cache.store(x, x.flip(0).contiguous(), torch.arange(64, device=gpu))
    table = torch.arange(4, dtype=torch.int32, device=gpu).view(2, 2)
    lengths, cu = torch.tensor([32, 20], dtype=torch.int32, device=gpu), torch.tensor([0, 3, 5], dtype=torch.int32, device=gpu)
    both = torch.randn(6, 2, 4, 64, generator=gen).half().to(gpu)
    q, free = both[:5, 0], both[:5, 1]
    want = cache.attend(q, table, lengths, cu_q=cu)
    for out in (both.view(6, -1)[:5, 1:257].unflatten(1, (4, 64)), both.view(6, -1)[:5, 255:511].unflatten(1, (4, 64)), both[1:, 0]):
        with pytest.raises(RuntimeError, match="share memory"):
            cache.attend(q, table, lengths, cu_q=cu, out=out)
    assert torch.equal(cache.attend(q, table, lengths, cu_q=cu, out=free), want)
    rows = torch.tensor([0, 32, 52], dtype=torch.int32, device=gpu)
    k, v = cache.load(table, rows, 52)
    buffer = torch.zeros(53, 4, 64, device=gpu).half()
    for v_out in (buffer[:52, :2], buffer[:52, 1:3], buffer[1:, :2]):
        with pytest.raises(RuntimeError, match="share memory"):
            cache.load(table, rows, 52, k_out=buffer[:52, :2], v_out=v_out)
    assert (buffer == 0).all()
    cache.load(table, rows, 52, k_out=buffer[:52, :2], v_out=buffer[1:, 2:])
    assert torch.equal(buffer[:52, :2], k) and torch.equal(buffer[1:, 2:], v)


def test_offsets_of_more_sequences_than_a_call_takes(gpu):
    from uniql_amd.attention import prompt_attention
    x = torch.zeros(8, 4, 64, dtype=torch.float16, device=gpu)
    for count, words in ((2 ** 32 + 2, "larger than a call"), (2 ** 30 + 2, "sizes")):
        with pytest.raises(RuntimeError, match=words):
            prompt_attention(x, x, x, torch.empty(count, dtype=torch.int32, device=gpu))
