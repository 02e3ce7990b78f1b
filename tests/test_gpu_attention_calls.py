"""The attention operators in a user's hands: calls in graphs, on several streams, of sizes that change, and what they
report, against the 64-bit forms of tests/attention_ref.py."""

import pytest

from tests import attention_ref as ref
from tests.test_gpu_attention import Pool, _check_decode, _check_prompt, ints, offsets_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def fresh():
    """A handle of its own, whose workspace has no size yet."""
    from voxwerk_b200 import Device
    with Device(0) as d:
        yield d


@pytest.mark.parametrize("prefixes", [[], [500]], ids=["own keys", "prefix"])
def test_captured_step_outlives_the_workspace_it_was_captured_with(fresh, prefixes):
    """A step is captured; eager calls that need more workspace follow; replays still give the formula's values."""
    import torch
    from voxwerk_b200 import KvBatch, KvPrefix, decode_attention, prompt_attention
    pool = Pool(700, 16, 2, 128, seed=21)
    lens = [700, 3, 450, 1200]
    table = pool.table(lens)
    ptable = pool.table(prefixes) if prefixes else None
    groups = [0, 3] if prefixes else ()
    prefix = KvPrefix(ptable, ints(prefixes), ints(groups)) if prefixes else None
    q = pool.normal(4, 4, 128)
    out = torch.full_like(q, 9.0)
    batch = KvBatch(table, ints(lens))
    prompt_lens = [2500, 900, 1100]
    prompt_table = pool.table(prompt_lens)
    pq = pool.normal(sum(prompt_lens) // 4, 4, 128)
    rows = [n // 4 for n in prompt_lens]
    pq = pq[:sum(rows)]
    big = KvBatch(prompt_table, ints(prompt_lens), ints(offsets_of(rows)))
    pout = torch.full_like(pq, 9.0)
    many = KvBatch(table[:1].expand(3000, table.shape[1]).contiguous(), ints([5] * 3000))
    mq, mout = pool.normal(3000, 4, 128), torch.empty((3000, 4, 128), dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    step = lambda: decode_attention(fresh, q, pool.cache, batch, out, prefix=prefix, stream=stream.cuda_stream)
    step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for _ in range(3):
        out.fill_(9.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        prompt_attention(fresh, pq, pool.cache, big, pout, stream=stream.cuda_stream)
        with torch.cuda.stream(stream):
            graph.replay()
        decode_attention(fresh, mq, pool.cache, many, mout, stream=stream.cuda_stream)
        out_of_the_way = torch.full((1 << 24,), float("nan"), device="cuda")   # takes what was freed
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        fresh.synchronize(stream.cuda_stream)
        del out_of_the_way
        _check_decode(pool, table, ptable, q, out, None, lens, prefixes, groups, 128 ** -0.5)
    _check_prompt(pool, prompt_table, pq, pout, None, rows, prompt_lens, 128 ** -0.5)
    del graph


def test_an_error_read_on_one_stream_leaves_calls_of_another_alone(device):
    """Prompts and steps run on one stream while another's calls fail and their errors are read."""
    import torch
    from voxwerk_b200 import KvBatch, KvPrefix, VwOutOfRange, decode_attention, prompt_attention, rope_append
    pool = Pool(1300, 16, 2, 128, seed=22)
    lens, prefixes = [40 + 37 * i for i in range(30)], [900]
    table, ptable = pool.table(lens), pool.table(prefixes)
    q = pool.normal(30, 4, 128)
    rows = [n // 2 for n in lens]
    pq = pool.normal(sum(rows), 4, 128)
    batch, prefix = KvBatch(table, ints(lens)), KvPrefix(ptable, ints(prefixes), ints([0, 30]))
    prompts = KvBatch(table, ints(lens), ints(offsets_of(rows)))
    outs = [(torch.full_like(q, 9.0), torch.full_like(pq, 9.0), torch.full_like(q, 9.0)) for _ in range(40)]
    bad = table[:1].clone()
    bad[0, 0] = 1300
    bad_batch = KvBatch(bad, ints([5]))
    bad_q, bad_k = pool.normal(1, 4, 128), pool.normal(1, 2, 128)
    bad_out = torch.empty_like(bad_q)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for step, prompt, alone in outs:
        decode_attention(device, q, pool.cache, batch, step, prefix=prefix, stream=b.cuda_stream)
        prompt_attention(device, pq, pool.cache, prompts, prompt, stream=b.cuda_stream)
        decode_attention(device, q, pool.cache, batch, alone, stream=b.cuda_stream)
        rope_append(device, bad_q, bad_k, bad_k, pool.cache, bad_batch, None, bad_out, stream=a.cuda_stream)
        with pytest.raises(VwOutOfRange, match="page"):
            device.synchronize(a.cuda_stream)
    device.synchronize(b.cuda_stream)
    first = outs[0]
    _check_decode(pool, table, ptable, q, first[0], None, lens, prefixes, [0, 30], 128 ** -0.5)
    _check_prompt(pool, table, pq, first[1], None, rows, lens, 128 ** -0.5)
    _check_decode(pool, table, None, q, first[2], None, lens, [], [], 128 ** -0.5)
    for other in outs[1:]:
        for x, y in zip(first, other):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16))


def test_a_call_that_waits_reports_an_enqueued_call_s_error(fresh):
    """Whichever call waits next: an attention call, or the sampler's."""
    import torch
    from voxwerk_b200 import (KvBatch, SamplingOptions, Segment, VwInvalidArgument, decode_attention, prompt_attention,
                              rope_append, sample_rows, vw_options)
    pool = Pool(20, 16, 2, 64, seed=23)
    table = pool.table([20, 30])
    q, k = pool.normal(2, 4, 64), pool.normal(2, 2, 64)
    out = torch.empty_like(q)
    good, bad = KvBatch(table, ints([20, 30])), KvBatch(table, ints([20, -1]))
    ids = torch.empty(2, dtype=torch.int32, device="cuda")
    segment = Segment(torch.randn((2, 64), device="cuda"), out_ids=ids)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for waits in (lambda: prompt_attention(fresh, q, pool.cache, good, out),
                  lambda: decode_attention(fresh, q, pool.cache, good, out),
                  lambda: rope_append(fresh, q, k, k, pool.cache, good, None, out),
                  lambda: sample_rows(fresh, [segment], [vw_options(SamplingOptions.greedy())])):
        waits()
        decode_attention(fresh, q, pool.cache, bad, out, stream=stream.cuda_stream)
        stream.synchronize()
        with pytest.raises(VwInvalidArgument, match="kv_lens"):
            waits()
        waits()


def test_prompt_with_fewer_rows_than_sequences(device):
    """Without q_offsets row s is sequence s; sequences past the last row have none, which is no error."""
    import torch
    from voxwerk_b200 import KvBatch, prompt_attention
    pool = Pool(60, 16, 2, 64, seed=24)
    lens = [70, 5, 33, 0, 90]
    table = pool.table(lens)
    for rows in (1, 2, 3, 5):
        q = pool.normal(rows, 4, 64)
        out, ls = torch.full_like(q, 9.0), torch.full((rows, 4), 9.0, device="cuda")
        torch.cuda.synchronize()
        prompt_attention(device, q, pool.cache, KvBatch(table, ints(lens)), out, lse=ls)
        _check_prompt(pool, table, q, out, ls, [1] * rows, lens[:rows], 0.125)


@pytest.mark.parametrize("n,rows", [(2, 20), (70, 500), (300, 4)])
def test_append_reports_row_offsets_that_do_not_fit(device, n, rows):
    """Offsets past the rows, below zero or descending are reported, as by the attention calls; the rows of a sequence
    whose own offsets do not fit are left alone."""
    import torch
    from voxwerk_b200 import KvBatch, VwInvalidArgument, rope_append
    pool = Pool(8 * n + 1, 16, 1, 64, seed=25)
    lens = [100] * n
    table = pool.table(lens, fill=False)
    q, k = pool.normal(rows, 2, 64), pool.normal(rows, 1, 64)
    q_out = torch.full_like(q, 9.0)
    good = [rows * s // n for s in range(n + 1)]
    past, below, descending = list(good), list(good), list(good)
    past[n] = rows + 1
    below[0] = -3
    descending[n // 2 + 1] = good[n // 2] - 1
    torch.cuda.synchronize()
    for offsets, alone in ((past, [n - 1]), (below, [0]), (descending, [])):
        q_out.fill_(9.0), pool.k.fill_(float("nan"))
        torch.cuda.synchronize()
        with pytest.raises(VwInvalidArgument, match="q_offsets"):
            rope_append(device, q, k, k, pool.cache, KvBatch(table, ints(lens), ints(offsets)), None, q_out)
        for s in alone:
            assert bool((q_out[max(offsets[s], 0):min(offsets[s + 1], rows)] == 9.0).all()), "rows were written"
            assert bool(torch.isnan(pool.k[table[s].long()]).all()), "keys were written"
        others = [s for s in range(n) if s not in alone and offsets is not descending]
        for s in others:
            assert torch.equal(q_out[offsets[s]:offsets[s + 1]], q[offsets[s]:offsets[s + 1]])
    rope_append(device, q, k, k, pool.cache, KvBatch(table, ints(lens), ints(good)), None, q_out)
    assert torch.equal(q_out, q)


def _us(call, times=5):
    """The shortest of some calls, on the device."""
    import torch
    best = float("inf")
    for _ in range(times):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        torch.cuda.synchronize()
        best = min(best, start.elapsed_time(end) * 1e3)
    return best


@pytest.mark.parametrize("n,heads,kv", [(256, 16, 2), (4096, 64, 1)])
def test_prompts_after_very_different_numbers_of_keys(device, n, heads, kv):
    """Many short prompts and one that continues 8000 cached keys: right, and no slower than the two apart.  The long one's
    block is one CTA's work, 63 key tiles of at most 2.3 us each; twice the sum, for the timing's sake."""
    import torch
    from voxwerk_b200 import KvBatch, prompt_attention
    pool = Pool(n + 40, 256, kv, 64, seed=26)
    rows = [1 + i % 3 for i in range(n)]
    short = list(rows)
    mixed = list(rows)
    mixed[n // 3] += 8000
    stream = torch.cuda.Stream()

    def batch(total, new):
        table = pool.table(total)
        q = pool.normal(sum(new), heads, 64)
        out = torch.full_like(q, 9.0)
        b = KvBatch(table, ints(total), ints(offsets_of(new)))
        torch.cuda.synchronize()
        return (table, q, out), lambda: prompt_attention(device, q, pool.cache, b, out, stream=stream.cuda_stream)

    (table, q, out), call = batch(mixed, rows)
    with torch.cuda.stream(stream):
        together = _us(call)
        _check_prompt(pool, table, q, out, None, rows, mixed, 0.125)
        pool.free = list(range(n + 40))
        apart = _us(batch(short, rows)[1]) + 63 * 2.3
    device.synchronize(stream.cuda_stream)
    assert together < 2 * apart, f"{together:.0f} us together, {apart:.0f} us apart"


@pytest.mark.parametrize("how", ["no stream", "no stream, on a side stream", "default stream"])
def test_inputs_that_the_current_stream_still_makes(device, how):
    """A call is in order with the kernels that make its inputs and with those that read its outputs."""
    import contextlib
    import torch
    from voxwerk_b200 import KvBatch, decode_attention, prompt_attention, rope_append
    pool = Pool(40, 16, 2, 64, seed=27)
    lens = [100, 60, 33]
    table = pool.table(lens)
    batch, prompts = KvBatch(table, ints(lens)), KvBatch(table, ints(lens), ints([0, 40, 60, 90]))
    made, pmade, kmade = pool.normal(3, 4, 64), pool.normal(90, 4, 64), pool.normal(3, 2, 64)
    q, pq, k = torch.zeros_like(made), torch.zeros_like(pmade), torch.zeros_like(kmade)
    out, pout, q_out = torch.full_like(q, 9.0), torch.full_like(pq, 9.0), torch.full_like(q, 9.0)
    side = torch.cuda.Stream()
    work = torch.randn((4096, 4096), device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side) if "side" in how else contextlib.nullcontext():
        stream = 0 if how == "default stream" else None
        if stream == 0:
            assert torch.cuda.current_stream().cuda_stream == 0
        for _ in range(10):
            work = torch.relu(work @ work) * 1e-4      # some milliseconds
        q.copy_(made), pq.copy_(pmade), k.copy_(kmade)
        decode_attention(device, q, pool.cache, batch, out, stream=stream)
        prompt_attention(device, pq, pool.cache, prompts, pout, stream=stream)
        got, pgot = out.clone(), pout.clone()
        q.zero_()
        for _ in range(10):
            work = torch.relu(work @ work) * 1e-4
        q.copy_(made)
        rope_append(device, q, k, k, pool.cache, batch, None, q_out, stream=stream)
        written = q_out.clone()
    torch.cuda.synchronize()
    device.synchronize()
    assert torch.equal(written, made)
    last = [n - 1 for n in lens]
    assert all(torch.equal(pool.k[table[s, n // 16].long(), n % 16], kmade[s]) for s, n in enumerate(last))
    keep = Pool(40, 16, 2, 64, seed=27)        # the cache before the last call wrote to it
    assert torch.equal(keep.table(lens), table)
    _check_decode(keep, table, None, made, got, None, lens, [], [], 0.125)
    _check_prompt(keep, table, pmade, pgot, None, [40, 20, 30], lens, 0.125)


def test_voices_that_the_current_stream_still_makes():
    """The example's prompts may come straight from kernels that are still running, and be dropped at once."""
    import torch
    from examples.voice_decoder import VoiceDecoder
    from voxwerk_b200 import Device
    with Device(0) as device:
        make = lambda: VoiceDecoder(device, [37, 80], [0, 1, 1], 4, layers=1, hidden=256, heads=4, kv_heads=2, dim=64,
                                    inner=512, vocab=512, seed=3)
        a, b = make(), make()
        x = torch.randn((117, 256), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
        work = torch.randn((4096, 4096), device="cuda")
        torch.cuda.synchronize()
        want = a.read_voices(x)
        a.check()
        for _ in range(10):
            work = torch.relu(work @ work) * 1e-4      # some milliseconds
        made = torch.zeros_like(x)
        made.copy_(x)
        got = b.read_voices(made)
        del made
        reused = [torch.full_like(x, float("nan")) for _ in range(4)]
        b.check()
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
        del reused


@pytest.mark.parametrize("scale", [0.0, -0.07, -1.5, 1e-6])
def test_scales_of_every_sign(device, scale):
    """Also those under which every key weighs the same, or the least alike the most."""
    from tests.test_gpu_attention import _decode, _prompt
    lens = [1, 0, 70, 33, 129, 400]
    _decode(device, 4, 2, 128, 16, lens, seed=28, scale=scale)
    _decode(device, 6, 2, 64, 32, lens, [300, 17], [0, 4, 6], seed=29, scale=scale)
    _decode(device, 34, 2, 128, 64, lens, [300], [1, 5], seed=30, scale=scale)
    _prompt(device, 4, 2, 128, 16, [1, 70, 0, 33, 129], [0, 0, 5, 100, 3], seed=31, scale=scale)
    _prompt(device, 8, 1, 64, 64, [5, 64], [3000, 500], seed=32, scale=scale)


@pytest.mark.parametrize("where", ["own keys", "prefix"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_decode_keys_that_are_not_finite(device, where, dim, page):
    """A key of NaN makes the rows that see it NaN; one whose score is -inf has no weight, +inf leaves nothing finite.  Rows
    that do not see it do not notice."""
    import torch
    from voxwerk_b200 import KvBatch, KvPrefix, decode_attention
    lens, prefixes, groups = [200, 90, 75, 300, 0], [500, 130], [0, 3, 5]
    for bad, place in ((float("nan"), 70), (float("inf"), 70), (float("inf"), 0), (-float("inf"), 74)):
        pool = Pool(120, page, 2, dim, seed=33)
        table, ptable = pool.table(lens), pool.table(prefixes)
        row, sees = (table[2], [2]) if where == "own keys" else (ptable[0], [0, 1, 2])
        at = row.long()[place // page], place % page
        pool.k[at[0], at[1], :, 3] = bad       # one dim: the score is bad times the query's sign
        q = pool.normal(5, 4, dim)
        out, ls = torch.full_like(q, 9.0), torch.full((5, 4), 9.0, device="cuda")
        torch.cuda.synchronize()
        decode_attention(device, q, pool.cache, KvBatch(table, ints(lens)), out, lse=ls,
                         prefix=KvPrefix(ptable, ints(prefixes), ints(groups)))
        shared = [tuple(ref.keys_of(c, ptable[g], p) for c in (pool.k, pool.v)) for g, p in enumerate(prefixes)]
        for s, n in enumerate(lens):
            k, v = (ref.keys_of(c, table[s], n) for c in (pool.k, pool.v))
            k, v = torch.cat([shared[s > 2][0], k]), torch.cat([shared[s > 2][1], v])
            if s in sees:
                keep = torch.isfinite(k).flatten(1).all(1)
                assert int((~keep).sum()) == 1
                k, v = k[keep], v[keep]
            want, lse, bound, lse_bound = ref.attend(q[s:s + 1], k, v, dim ** -0.5)
            if s not in sees:
                ref.check(out[s:s + 1], want, bound, f"sequence {s}")
                ref.check(ls[s:s + 1], lse, lse_bound, f"sequence {s} lse")
                continue
            for h in range(4):
                if bad != bad or float(q[s, h, 3]) * bad > 0:
                    assert bool(torch.isnan(out[s, h].float()).all()), f"sequence {s} head {h} of a key of {bad}"
                    assert not bool(torch.isfinite(ls[s, h]))
                else:
                    ref.check(out[s:s + 1, h], want[:, h], bound[:, h], f"sequence {s} head {h}")
                    ref.check(ls[s:s + 1, h], lse[:, h], lse_bound[:, h], f"sequence {s} head {h} lse")


def test_prompts_of_many_lengths_behind_many_numbers_of_keys(device):
    """More sequences than a warp has lanes, their blocks on many levels of key counts with gaps between."""
    from tests.test_gpu_attention import _prompt
    n = 90
    _prompt(device, 8, 2, 64, 64, [1 + (29 * i) % 50 for i in range(n)], [(613 * i) % 3000 for i in range(n)], seed=34)
    _prompt(device, 16, 1, 128, 16, [(7 * i) % 40 for i in range(200)], [(i % 3) * 800 for i in range(200)], seed=35)
