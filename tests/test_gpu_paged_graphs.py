"""A PagedCache whose steps are captured in a graph: what the host knows of it
after replays."""
import pytest
import torch

from nativebit_amd import paged
from nativebit_amd.model import ModelConfig, random_packed_model

pytestmark = pytest.mark.gpu


def test_lists_after_replays(dev):
    """Replays between steps from lists: lengths and blocks that they took count."""
    cfg = ModelConfig(vocab_size=100, n_layers=1, n_embd=64, n_head=1, ffn_hidden=128, context_len=200)
    model = random_packed_model(cfg, seed=1, device=dev)
    c = paged.PagedCache(model, 5, 2)
    ones, idx = torch.ones(2, dtype=torch.int32, device=dev), torch.ones(1, 2, dtype=torch.int64, device=dev)

    def one():
        c.step(ones, n_tokens=2)
        model(idx, kv_caches=c)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        one()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        one()
    c.step([100, 20])       # 101 and 21 tokens, three blocks
    assert c.lens.tolist() == [101, 21]
    for _ in range(43):
        g.replay()
    assert c.lens.tolist() == [144, 64] and c.state.tolist() == [1, 0]
    with pytest.raises(ValueError, match="max_len"):
        c.step([57, 0])     # (the host saw 101 last)
    with pytest.raises(ValueError, match="blocks"):
        c.step([49, 1])     # two blocks, one is free
    c.step([48, 1])
    g.replay()
    assert c.lens.tolist() == [192, 66] and c.state.tolist() == [0, 1]   # no block for the 193rd
    c.release([1])
    c.step([0, 120])        # both blocks that it had at its end
    assert c.lens.tolist() == [192, 120] and c.state.tolist() == [0, 0]
    with pytest.raises(ValueError, match="blocks"):
        c.step([0, 60])
