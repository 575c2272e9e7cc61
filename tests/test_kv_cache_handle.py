"""The native handle of a cache's tensors belongs to the tensors that the module holds at the call (no GPU needed)."""
import pytest
import torch

from uniql_amd.quantize.quant_kv_cache import W4KVCache

NAMES = ["k_codes", "k_scales", "v_codes", "v_scales"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("how", ["assigned", "registered", "written", "a view of itself"])
def test_a_replaced_tensor_asks_for_a_new_handle(name, how):
    cache = W4KVCache(4, 16, 2, 64)
    handle = cache._native()
    assert cache._native() is handle
    new = getattr(cache, name).clone()
    if how == "assigned":
        setattr(cache, name, new)
    elif how == "registered":
        cache.register_buffer(name, new, persistent=False)
    elif how == "written":
        cache._buffers[name] = new
    else:
        cache._buffers[name] = getattr(cache, name)[:2]
    other = cache._native()
    assert other is not handle and cache._native() is other


def test_a_call_with_other_tensors_for_its_time_only():
    class Holder(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.cache = W4KVCache(4, 16, 2, 64)

        def forward(self):
            return self.cache._native()

    holder = Holder()
    mine = holder()
    theirs = torch.func.functional_call(holder, {"cache.k_codes": holder.cache.k_codes.clone()}, ())
    assert theirs is not mine
    assert holder() is not theirs      # the module has its own tensors again


def test_other_widths_ask_for_a_new_handle():
    cache = W4KVCache(4, 16, 2, 64)
    handle = cache._native()
    cache.head_dim = 60
    assert cache._native() is not handle


def test_a_moved_module_keeps_nothing_of_the_old_tensors():
    import gc
    import weakref
    cache = W4KVCache(4, 16, 2, 64)
    cache._native()
    old = weakref.ref(cache.k_scales.untyped_storage())
    cache.to(torch.float32)      # floating-point tensors are replaced
    gc.collect()
    assert "_handle" not in cache.__dict__ and old() is None
