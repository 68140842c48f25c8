"""The paged streaming decoder against the ring-cache streaming decoder: each
stream, whatever it shares its steps with, comes out as if it ran alone."""
import pytest
import torch

from mimi_chain import MimiChainConfig, PagedStreamingDecoder, StreamingDecoderChain, rope_tables, synthetic_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_paged_decoder_matches_one_stream_at_a_time(cuda, dtype, graph):
    cfg = MimiChainConfig(d_model=128, num_heads=2, num_layers=2, dim_feedforward=256, max_seq_len=64, context=20)
    w = synthetic_weights(cfg, dtype, cuda, seed=1)
    cos, sin = rope_tables(cfg, dtype, cuda)
    streams, cap = 3, 8
    paged = PagedStreamingDecoder(cfg, w, cos, sin, streams, pages=14, token_cap=cap, page_size=8, max_new=1)
    rings = [StreamingDecoderChain(cfg, w, cos, sin, 1, mask="absolute") for _ in range(streams)]
    x, new = torch.zeros(cap, cfg.d_model, dtype=dtype, device=cuda), torch.zeros(streams, dtype=torch.int64, device=cuda)
    if graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            paged.step(x, new)
        torch.cuda.current_stream().wait_stream(side)
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            out = paged.step(x, new)
    g = torch.Generator().manual_seed(2)
    for step in range(45):
        # Stream 0 always runs, 1 comes late, 2 pauses now and then; 1 ends at step 30 and begins anew at 33.
        active = [0] + ([1] if step >= 7 and not 30 <= step < 33 else []) + ([2] if step % 5 else [])
        frames = torch.randn(len(active), cfg.d_model, generator=g).to(dtype)
        x.zero_()
        x[:len(active)] = frames.to(cuda)
        new.copy_(torch.tensor([1 if i in active else -1 if i == 1 and step == 30 else 0 for i in range(streams)]))
        if graph:
            cg.replay()
        else:
            out = paged.step(x, new)
        assert int(paged.err_flag) == 0
        if step == 30:
            rings[1].reset()
        for row, i in enumerate(active):
            ref = rings[i].step(x[row].view(1, 1, -1)).view(-1).float()
            # Both evaluate one formula in sums of up to 256 terms, some 20 one behind the other:
            # 20 * 4 sqrt(256) * 2^-24 relative in f32. In bf16 the rings round each product of the rotation, the
            # scores and the weights, here only the operands: about six roundings of 2^-8 a layer on the branches,
            # whose share of the residual stream the layer scales (below 0.1) keep under a tenth.
            tol = 8e-5 if dtype == torch.float32 else 2 * 6 * 2.0 ** -8 * 0.2 + 2 * 2.0 ** -8
            assert (out[row].float() - ref).abs().max() <= tol * ref.abs().max(), (step, i)
    assert paged.lens.tolist() == [45, 12, 36]


def test_paged_decoder_prompt_then_frames(cuda):
    """A stream's first frames at once give what they give one at a time."""
    cfg = MimiChainConfig(d_model=128, num_heads=2, num_layers=2, dim_feedforward=256, max_seq_len=64, context=20)
    w = synthetic_weights(cfg, torch.float32, cuda, seed=1)
    cos, sin = rope_tables(cfg, torch.float32, cuda)
    frames = torch.randn(40, cfg.d_model, generator=torch.Generator().manual_seed(5)).to(cuda)
    one, many = (PagedStreamingDecoder(cfg, w, cos, sin, 1, pages=6, token_cap=n, page_size=8) for n in (1, 40))
    want = torch.cat([one.step(frames[i:i + 1], torch.ones(1, dtype=torch.int64, device=cuda)) for i in range(40)])
    got = many.step(frames, torch.full((1,), 40, dtype=torch.int64, device=cuda))
    assert int(one.err_flag) == 0 and int(many.err_flag) == 0
    assert (got - want).abs().max() <= 8e-5 * want.abs().max()
    # A step that does not fit leaves the stream as it was.
    many.step(frames, torch.full((1,), 40, dtype=torch.int64, device=cuda))
    assert int(many.err_flag) != 0 and many.lens.tolist() == [40]
