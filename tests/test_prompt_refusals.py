"""CPU-only: calls around the prompt operators that would have given a wrong result."""
import pytest
import torch


@pytest.mark.parametrize("queries", [1, 7, 19])
def test_rows_of_no_query_do_not_seed_a_ring(queries):
    """All rows for a prompt shorter than the ring, zeros behind its own: they would count as queries."""
    from hqekv_b200.model.public_func import last_attn_weights
    ring = last_attn_weights(last_length=20)
    ring.set_max_length(400)
    with pytest.raises(ValueError, match="positions"):
        ring.seed(torch.zeros(20, queries, dtype=torch.float16))
    assert ring.weights is None and (ring.next_line, ring.kv_seq_len) == (0, 0)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ring.seed(torch.zeros(queries, queries, dtype=torch.float16))
