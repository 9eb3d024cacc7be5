"""What the modules with norms of queries and keys refuse before they touch a GPU."""
import pytest
import torch

from nmtgminor_amd.modules import window_attention as wa

BF16 = torch.bfloat16


@pytest.fixture
def host_projections(monkeypatch):
    """The projections alone on the CPU, so that what stands behind them decides."""
    monkeypatch.setattr(wa, "linear_function", torch.nn.functional.linear)


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("learned", ["q_norm_weight", "k_norm_weight"])
def test_norm_weights_that_learn_are_no_part_of_decoding_from_a_cache(host_projections, learned, first):
    """Keys in the cache have no gradient: neither a prompt nor a step leaves it out silently."""
    m = wa.WindowSelfMultiheadAttn(128, 2, window=4, qk_norm=True).bfloat16().requires_grad_(False)
    getattr(m, learned).requires_grad_()
    cache = m.make_cache(1, 8)
    cache.longest = 0 if first else 3
    pos = torch.zeros(16, 64), torch.zeros(16, 64)
    with pytest.raises(RuntimeError, match="no gradient, call it under torch.no_grad"):
        m(torch.zeros(3 if first else 1, 1, 128, dtype=BF16), cache=cache, pos_emb=pos)
    assert cache.lengths.tolist() == [0]
