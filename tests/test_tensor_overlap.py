"""Whether tensors of heads share memory, against the sets of their elements (no GPU needed)."""
import random

import torch

from uniql_amd import _capi


def elements(t):
    return (t.storage_offset() + sum(torch.arange(n).view([-1 if i == a else 1 for i in range(3)]) * s
                                     for a, (n, s) in enumerate(zip(t.shape, t.stride())))).flatten().tolist()


def drawn(rng, buffer):
    rows, heads, width = rng.randint(1, 6), rng.randint(1, 5), rng.randint(1, 6)
    head = rng.choice((width, width, width + rng.randint(0, 4), rng.randint(0, 12), 40))
    row = rng.choice((heads * head, heads * head + rng.randint(0, 9), rng.randint(0, 40), 24, 48, width))
    return buffer.as_strided((rows, heads, width), (row, head, 1), rng.randint(0, 150))


def test_two_tensors():
    host, rng = _capi.host(), random.Random(1)
    buffer, found = torch.zeros(1400).half(), [0, 0]
    for _ in range(60000):
        a, b = drawn(rng, buffer), drawn(rng, buffer)
        want = not set(elements(a)).isdisjoint(elements(b))
        found[want] += 1
        assert host.share_memory(a, b) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
    assert min(found) > 10000


def test_neighbours_in_a_fused_buffer():
    """column ranges and interleaved heads of one buffer, rows one after the other or in turn"""
    host = _capi.host()
    x = torch.zeros(50, 4 * 24 + 2 * 24).half()
    q, k = x[:, :96].view(50, 4, 24), x[:, 96:].view(50, 2, 24)
    assert not host.share_memory(q, k) and not host.share_memory(k, q) and host.share_memory(q, q)
    assert host.share_memory(x[:, 1:97].view(50, 4, 24), q) and host.share_memory(x[:, 90:138].view(50, 2, 24), q)
    y = torch.zeros(50, 4, 3 * 24).half()
    parts = y.split(24, dim=2)
    for i in range(3):
        for j in range(3):
            assert host.share_memory(parts[i], parts[j]) == (i == j)
    assert not host.share_memory(y[::2], y[1::2]) and not host.share_memory(y[:25], y[25:]) and host.share_memory(y[:26], y[25:])
    assert not host.share_memory(y[::2], y[1::4]) and host.share_memory(y[::2], y[::4])
    assert not host.share_memory(y[:0], y) and not host.share_memory(y, torch.zeros_like(y))


def test_a_tensor_and_itself():
    host, rng = _capi.host(), random.Random(2)
    buffer, found = torch.zeros(1400).half(), [0, 0]
    for _ in range(30000):
        a = drawn(rng, buffer)
        own = elements(a)
        want = len(set(own)) < len(own)
        found[want] += 1
        assert host.overlaps_itself(a) == want, (a.shape, a.stride())
    assert min(found) > 5000
    assert not host.overlaps_itself(torch.zeros(3, 5, 7).half().transpose(0, 1))
    assert not host.overlaps_itself(buffer.as_strided((4, 1, 8), (8, 0, 1)))
    assert host.overlaps_itself(buffer.as_strided((4, 3, 8), (8, 8, 1))) and host.overlaps_itself(buffer.as_strided((4, 3, 8), (0, 8, 1)))
