"""Sampler calls captured into a CUDA graph keep their buffers and their options, whatever eager calls follow."""

import pytest

pytestmark = pytest.mark.gpu


def test_captured_calls_keep_their_logits_and_options():
    import torch
    from voxwerk_b200 import VW_ROWS_SUB, Device, SamplingOptions, Segment, head_sample, sample_rows, vw_options
    g = torch.Generator(device="cuda").manual_seed(5)
    rows, vocab = 40, 2048
    hidden = torch.randn((rows, 64), generator=g, device="cuda").to(torch.bfloat16)
    weight = torch.randn((vocab, 64), generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.randn((rows, vocab), generator=g, device="cuda")
    uniforms = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    ids, head_ids = (torch.full((rows,), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    each = torch.arange(rows, dtype=torch.int32, device="cuda")
    table = lambda at: [vw_options(SamplingOptions(top_k=0, temperature=at + 0.02 * i)) for i in range(rows)]
    segment = Segment(logits, kind=VW_ROWS_SUB, out_ids=ids, uniforms=uniforms, opt_index=each)
    head = Segment(None, kind=VW_ROWS_SUB, vocab=vocab, out_ids=head_ids, uniforms=uniforms)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with Device(0) as device:
        def step(stream):
            sample_rows(device, [segment], table(0.4), stream=stream)
            head_sample(device, hidden, weight, head, table(0.9)[:1], stream=stream)
        step(stream.cuda_stream)
        device.synchronize(stream.cuda_stream)
        want = ids.clone(), head_ids.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(stream.cuda_stream)
        n = 6000
        many = Segment(None, kind=VW_ROWS_SUB, vocab=vocab, out_ids=torch.empty(n, dtype=torch.int32, device="cuda"),
                       uniforms=torch.rand(n, generator=g, device="cuda", dtype=torch.float64))
        wide = torch.randn((n, 64), generator=g, device="cuda").to(torch.bfloat16)
        torch.cuda.synchronize()
        head_sample(device, wide, weight, many, table(0.9)[:1], stream=stream.cuda_stream)
        sample_rows(device, [segment], table(4.0), stream=stream.cuda_stream)
        device.synchronize(stream.cuda_stream)
        assert not torch.equal(ids, want[0]), "the other table gives other ids"
        takes_what_was_freed = torch.full((1 << 24,), float("nan"), device="cuda")
        ids.fill_(-1), head_ids.fill_(-1)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        device.synchronize(stream.cuda_stream)
        assert torch.equal(ids, want[0]) and torch.equal(head_ids, want[1])
        del graph, takes_what_was_freed
