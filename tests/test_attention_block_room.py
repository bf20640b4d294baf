"""The example's batch at the end of its room: what lies past it has no place, and no look-up leaves the table."""
import pytest

torch = pytest.importorskip("torch")
from test_attention_block import example  # noqa: E402,F401


def test_steps_past_the_room_have_no_slot(example):  # noqa: F811
    seqs = example.Sequences(3, 32, 16, torch.device("cpu"))
    seqs.grow([31, 5, 30])
    last = None
    for n in range(4):
        pos, slots, _ = seqs.step()
        for i, first in enumerate((31, 5, 30)):
            p = min(first + n, 32)
            assert pos[i] == p and slots[i] == (int(seqs.table[i, p // 16]) * 16 + p % 16 if p < 32 else -1)
    assert seqs.kv_len.tolist() == [32, 9, 32]
    # prompts after steps that the host has not counted
    pos, slots, starts = seqs.grow([1, 20, 0])
    assert starts.tolist() == [0, 1, 21, 21]
    assert slots[0] == -1 and bool((slots[1:] >= 0).all()) and seqs.kv_len.tolist() == [32, 29, 32]


@pytest.mark.gpu
def test_a_graph_replayed_past_the_room(example):  # noqa: F811
    """Full sequences attend to what they hold, bit for bit the same at every further step of the same input."""
    dev, hidden = torch.device("cuda:0"), 512
    torch.manual_seed(3)
    block = example.synthetic_block(hidden, 8, 2, 64, "f16", dev)
    seqs = example.Sequences(2, 16, 16, dev)
    cache = example.new_cache(seqs.pages, 2, 16, 64, "f16", dev)
    h = example.pkg.synthetic_activations(20 * hidden, 5, device=dev).view(-1, hidden)
    block(h, cache, seqs, seqs.grow([14, 6]), 14, 16)
    step = example.pkg.synthetic_activations(2 * hidden, 6, device=dev).view(-1, hidden)
    graph, out = example.decode_graph(block, cache, seqs, step, seqs.room)
    outs = []
    for _ in range(13):
        graph.replay()
        torch.cuda.synchronize()
        outs.append(out.clone())
    assert seqs.kv_len.tolist() == [16, 16]
    kept = cache.k_pages.clone()
    graph.replay()
    assert torch.equal(cache.k_pages, kept) and torch.equal(out, outs[-1]) and torch.equal(outs[-1], outs[-2])
