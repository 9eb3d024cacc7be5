"""What the modules with norms of queries and keys refuse before they touch a GPU."""
import pytest
import torch

from nmtgminor_amd.modules import linear_attention as la
from nmtgminor_amd.modules import quantized_cache as qc
from nmtgminor_amd.modules import window_attention as wa

BF16 = torch.bfloat16


@pytest.fixture
def host_projections(monkeypatch):
    """The projections alone on the CPU, so that what stands behind them decides."""
    for module in (wa, la):
        monkeypatch.setattr(module, "linear_function", torch.nn.functional.linear)


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


def test_positions_behind_the_tables_are_refused_where_the_host_knows_of_them(host_projections, monkeypatch):
    """What is accepted ends at the kernels, which have no CPU path."""
    monkeypatch.setattr(qc, "kv_cache_write", lambda *args: None)
    pos = torch.zeros(6, 64), torch.zeros(6, 64)
    rows = lambda t: torch.zeros(t, 2, 128, dtype=BF16)                                # noqa: E731
    beyond, accepted = "of tables of 6 rows", "device memory"
    heads = torch.zeros(4, 2, 2, 64, dtype=BF16)
    with torch.no_grad():
        m = la.LinearSelfMultiheadAttn(128, 2).bfloat16()
        state = la.LinearAttnState(2, 2, 64, device="cpu")
        for t, lengths, said in ((6, None, accepted), (7, None, beyond), (7, torch.tensor([6, 2]), accepted)):
            with pytest.raises(RuntimeError, match=said):
                m(rows(t), lengths, state=state, pos_emb=pos)
        m = wa.WindowSelfMultiheadAttn(128, 2, window=4, qk_norm=True).bfloat16()
        cache = m.make_cache(2, 32)
        for t, lengths, said in ((6, None, accepted), (7, None, beyond), (7, torch.tensor([6, 2]), accepted)):
            with pytest.raises(RuntimeError, match=said):
                m(rows(t), lengths, cache=cache, pos_emb=pos)
        cache.append(heads, heads)
        for t, said in ((2, accepted), (3, beyond)):
            with pytest.raises(RuntimeError, match=said):
                m(rows(t), cache=cache, pos_emb=pos)
        # sequences may be shorter than what was appended
        cache.append(heads, heads, torch.tensor([4, 0]))
        assert (cache.shortest, cache.longest) == (4, 8)
        with pytest.raises(RuntimeError, match=accepted):
            m(rows(2), cache=cache, pos_emb=pos)
        # begun again
        cache.longest = 0
        cache.lengths.zero_()
        with pytest.raises(RuntimeError, match=accepted):
            m(rows(6), cache=cache, pos_emb=pos)
        cache.append(heads, heads)
        assert (cache.shortest, cache.longest) == (4, 4)
