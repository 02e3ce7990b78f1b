"""The operators together, as the example runs them: prompts read once, steps over shared prefixes, eager and in a graph."""

import pytest

pytestmark = pytest.mark.gpu

VOICES, VOICE_OF = [37, 80], [0, 0, 1, 1, 1]


@pytest.fixture
def make():
    import torch
    from examples.voice_decoder import VoiceDecoder
    from voxwerk_b200 import Device
    with Device(0) as device:
        def build():
            d = VoiceDecoder(device, VOICES, VOICE_OF, 20, layers=2, hidden=256, heads=4, kv_heads=2, dim=64, inner=512,
                             vocab=512, seed=3)
            g = torch.Generator().manual_seed(4)
            x = torch.randn((sum(VOICES), 256), generator=g).to(torch.bfloat16).cuda()
            torch.cuda.synchronize()
            return d, d.read_voices(x)
        yield build


def test_last_step_against_the_formulas(make):
    """The last layer's attention of a step, from the keys that the prompts and the steps put into the cache."""
    import torch
    from tests.attention_ref import attend, check, keys_of
    d, _ = make()
    for _ in range(18):      # past a page's end
        d.step()
    d.check()
    cache = d.layers[-1].cache
    assert d.kv_lens.tolist() == [18] * 5
    assert d.positions.tolist() == [VOICES[v] + 17 for v in VOICE_OF]
    for s, v in enumerate(VOICE_OF):
        k, val = (torch.cat([keys_of(c, d.prefix.page_table[v], VOICES[v]), keys_of(c, d.batch.page_table[s], 18)])
                  for c in (cache.k, cache.v))
        out, _, bound, _ = attend(d.q[s:s + 1], k, val, 64 ** -0.5)
        check(d.attended[s:s + 1], out, bound, f"sequence {s}")


def test_graph_replays_the_eager_steps(make):
    a, _ = make()
    b, _ = make()
    b.step()
    graph = b.capture()
    for _ in range(6):
        a.step()
    import torch
    with torch.cuda.stream(b.stream):
        for _ in range(5):
            graph.replay()
    a.check()
    b.check()
    assert torch.equal(a.attended.view(torch.int16), b.attended.view(torch.int16))
    assert torch.equal(a.ids, b.ids)
    del graph
