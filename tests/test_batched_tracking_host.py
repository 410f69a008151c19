"""What the batched hooks refuse before they touch a layer: no GPU is needed for layers that stay exact."""

import pytest
import torch

from turboquant_amd.integration import vllm as single
from turboquant_amd.integration.batched import install_batched_hooks
from turboquant_amd.integration.harness import MinimalRunner

SIZE = dict(n_layers=2, hidden=32, num_heads=4, num_kv_heads=2, ffn=32, vocab=10, batch=2, max_seq_len=32)


def runner(head_dim=64):
    return MinimalRunner(device="cpu", seed=5, head_dim=head_dim, **SIZE)


@pytest.fixture(autouse=True)
def mode_back():
    before = single.get_mode()
    yield
    single.set_mode(before)


class InForward:
    """A backend that writes its cache in forward()."""
    num_heads, num_kv_heads, head_size, scale = 4, 2, 64, 0.125

    def forward(self, *args):
        raise AssertionError("not called")


def refused(r, **kw):
    impls = [lay.attn.impl for lay in r.layers]
    single.set_mode("off")
    with pytest.raises(ValueError) as e:
        install_batched_hooks(r, r.num_blocks, mode="hybrid", **kw)
    assert single.get_mode() == "off" and not hasattr(r, "_tq_layer_states")
    assert all("forward" not in vars(i) and not hasattr(i, "_tq_layer_state") for i in impls)
    return str(e.value)


@pytest.mark.parametrize("which", [0, 1])
def test_exact_layers_of_a_backend_that_writes_its_cache_in_forward(which):
    r = runner()
    r.layers[which].attn.impl = InForward()
    assert "do_kv_cache_update" in refused(r, exact_layers=2)


@pytest.mark.parametrize("head_dim", [32, 96, 832])
def test_exact_layers_of_a_head_size_that_the_exact_cache_does_not_take(head_dim):
    assert "head_dim" in refused(runner(head_dim), exact_layers=2)


def test_exact_layers_that_are_taken():
    r = runner()
    assert len(install_batched_hooks(r, r.num_blocks, mode="hybrid", exact_layers=2)) == 2
    assert torch.is_tensor(r.kv_caches[0])
