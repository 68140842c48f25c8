"""The paged streaming decoder at the end of its lengths."""
import pytest
import torch

from mimi_chain import MimiChainConfig, PagedStreamingDecoder, rope_tables, synthetic_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_len", [None, 17])
def test_steps_past_the_last_position_change_nothing(xn, cuda, max_len):
    """A stream may have max_len positions, whole pages or not; a step that would pass them is refused whole."""
    cfg = MimiChainConfig(d_model=128, num_heads=2, num_layers=2, dim_feedforward=256, max_seq_len=20, context=12)
    w = synthetic_weights(cfg, torch.float32, cuda, seed=1)
    cos, sin = rope_tables(cfg, torch.float32, cuda)
    dec = PagedStreamingDecoder(cfg, w, cos, sin, 2, pages=8, token_cap=4, page_size=8, max_len=max_len)
    end = max_len or 20
    x = torch.randn(4, cfg.d_model, generator=torch.Generator().manual_seed(2)).to(cuda)
    new = lambda *v: torch.tensor(v, dtype=torch.int64, device=cuda)  # noqa: E731
    for _ in range(end // 4):
        dec.step(x, new(4, 0))
    for _ in range(end % 4):
        dec.step(x, new(1, 0))
    assert int(dec.err_flag) == 0 and dec.lens.tolist() == [end, 0]
    state = [t.clone() for t in (dec.k[0], dec.v[1], dec.table, dec.ring, dec.ring_state, dec.lens)]
    for step in ((1, 0), (1, 2), (4, 0)):
        dec.err_flag.zero_()
        dec.step(x, new(*step))
        assert int(dec.err_flag) == xn.XN_DEVERR_FULL
        for a, b in zip(state, (dec.k[0], dec.v[1], dec.table, dec.ring, dec.ring_state, dec.lens)):
            assert torch.equal(a, b)
    # The other stream goes on, and the first one may end.
    dec.err_flag.zero_()
    dec.step(x, new(0, 3))
    dec.step(x, new(-1, 1))
    assert int(dec.err_flag) == 0 and dec.lens.tolist() == [0, 4]


def test_lengths_beyond_the_rotation_tables_are_refused(cuda):
    cfg = MimiChainConfig(d_model=128, num_heads=2, num_layers=1, dim_feedforward=256, max_seq_len=20, context=12)
    w = synthetic_weights(cfg, torch.float32, cuda, seed=1)
    cos, sin = rope_tables(cfg, torch.float32, cuda)
    with pytest.raises(ValueError, match="20"):
        PagedStreamingDecoder(cfg, w, cos, sin, 1, pages=8, token_cap=4, page_size=8, max_len=21)


def test_a_captured_step_past_the_last_position(xn, cuda):
    cfg = MimiChainConfig(d_model=128, num_heads=2, num_layers=1, dim_feedforward=256, max_seq_len=11, context=12)
    w = synthetic_weights(cfg, torch.float32, cuda, seed=1)
    cos, sin = rope_tables(cfg, torch.float32, cuda)
    dec = PagedStreamingDecoder(cfg, w, cos, sin, 1, pages=4, token_cap=4, page_size=8)
    x = torch.randn(4, cfg.d_model, generator=torch.Generator().manual_seed(2)).to(cuda)
    new = torch.zeros(1, dtype=torch.int64, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dec.step(x, new)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dec.step(x, new)
    for n, lens, flag in ((4, 4, 0), (4, 8, 0), (4, 8, 4), (3, 11, 0), (1, 11, 4), (-1, 0, 0), (2, 2, 0)):
        dec.err_flag.zero_()
        new.fill_(n)
        graph.replay()
        assert (int(dec.lens), int(dec.err_flag)) == (lens, flag), n
