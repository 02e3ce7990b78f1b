"""A decoder that speaks for many sequences in a few voices, on the attention operators and the head's sampler.

The shape is the talker's of Qwen3-TTS (src/Voxwerk/Talker/DecoderStack.cs:144-228): RMS norm, q/k/v projections, heads
normalised and turned, attention over the cache, output projection, gated MLP.  A voice's prompt goes through the layers
once (`read_voices`: rope_append, prompt_attention) and stays in the cache as the prefix of every sequence that speaks
with it; `step` (rope_append, decode_attention, head_sample) adds a token to each sequence and can be captured into a
CUDA graph.  The projections are plain library products.  Weights are random:

    python examples/voice_decoder.py [--sequences 64] [--voice-tokens 300 500] [--steps 50]
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from voxwerk_b200 import (VW_ROWS_SUB, Device, KvBatch, KvCache, KvPrefix, RopeTable, SamplingOptions, Segment,
                          decode_attention, head_sample, prompt_attention, rope_append, vw_options)

PAGE = 16


def _rms(x, weight):
    y = x.float()
    return (y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6) * weight).to(torch.bfloat16)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Layer:
    def __init__(self, hidden, heads, kv_heads, dim, inner, n_pages, g):
        def weight(rows, cols):
            return (torch.randn((rows, cols), generator=g) * cols ** -0.5).to(torch.bfloat16).cuda()
        self.qkv, self.o = weight((heads + 2 * kv_heads) * dim, hidden), weight(hidden, heads * dim)
        self.gate_up, self.down = weight(2 * inner, hidden), weight(hidden, inner)
        self.norm1, self.norm2 = torch.ones(hidden, device="cuda"), torch.ones(hidden, device="cuda")
        self.q_norm, self.k_norm = torch.ones(dim, device="cuda"), torch.ones(dim, device="cuda")
        self.cache = KvCache.empty(n_pages, PAGE, kv_heads, dim)


class VoiceDecoder:
    """`voice_of[s]` is sequence s's voice, in rising order; every sequence may hold `max_tokens` keys of its own.  All
    work is enqueued on `stream`; `check` waits for it and raises what the kernels reported."""

    def __init__(self, device, voice_lens, voice_of, max_tokens, layers=4, hidden=1024, heads=16, kv_heads=8, dim=128,
                 inner=2048, vocab=2048, seed=0):
        self.device, self.heads, self.kv_heads, self.dim = device, heads, kv_heads, dim
        self.n, self.stream = len(voice_of), torch.cuda.Stream()
        g = torch.Generator().manual_seed(seed)
        pages = [-(-n // PAGE) for n in voice_lens]
        own = -(-max_tokens // PAGE)
        self.layers = [Layer(hidden, heads, kv_heads, dim, inner, sum(pages) + self.n * own, g) for _ in range(layers)]
        self.embed = torch.randn((vocab, hidden), generator=g).to(torch.bfloat16).cuda()
        self.head = (torch.randn((vocab, hidden), generator=g) * hidden ** -0.5).to(torch.bfloat16).cuda()
        self.final_norm = torch.ones(hidden, device="cuda")
        self.rope = RopeTable.build(max(voice_lens) + max_tokens, dim, base=1e6)

        voice_table = torch.zeros((len(pages), max(pages)), dtype=torch.int32)
        for i, n in enumerate(pages):
            voice_table[i, :n] = sum(pages[:i]) + torch.arange(n, dtype=torch.int32)
        first = sum(pages)
        table = (first + torch.arange(self.n * own, dtype=torch.int32)).view(self.n, own)
        starts = [0]
        for n in voice_lens:
            starts.append(starts[-1] + n)
        group_offsets = [sum(v < i for v in voice_of) for i in range(len(voice_lens) + 1)]
        voice_table, lens = voice_table.cuda(), _ints(voice_lens)
        self.voices = KvBatch(voice_table, lens, _ints(starts))
        self.prefix = KvPrefix(voice_table, lens, _ints(group_offsets))
        self.kv_lens = torch.zeros(self.n, dtype=torch.int32, device="cuda")
        self.positions = _ints([voice_lens[v] - 1 for v in voice_of])
        self.batch = KvBatch(table.cuda(), self.kv_lens)
        self.ids = torch.zeros(self.n, dtype=torch.int32, device="cuda")
        self.q = torch.empty((self.n, heads, dim), dtype=torch.bfloat16, device="cuda")
        self.attended = torch.empty_like(self.q)
        self.segment = Segment(None, kind=VW_ROWS_SUB, vocab=vocab, out_ids=self.ids)
        self.options = [vw_options(SamplingOptions.greedy())]
        torch.cuda.synchronize()      # the stream starts behind the set-up

    def _layers(self, x, batch, q, out, attend, positions=None):
        for layer in self.layers:
            h, k = self.heads, self.kv_heads
            qkv = (_rms(x, layer.norm1) @ layer.qkv.T).view(x.shape[0], h + 2 * k, self.dim)
            rope_append(self.device, qkv[:, :h], qkv[:, h:h + k], qkv[:, h + k:], layer.cache, batch, self.rope, q,
                        q_norm=layer.q_norm, k_norm=layer.k_norm, positions=positions, stream=self.stream.cuda_stream)
            attend(layer.cache)
            x = x + out.view(x.shape[0], -1) @ layer.o.T
            gate, up = (_rms(x, layer.norm2) @ layer.gate_up.T).chunk(2, dim=-1)
            x = x + (torch.nn.functional.silu(gate) * up) @ layer.down.T
        return x

    def read_voices(self, x):
        """x [sum(voice_lens), hidden] bfloat16: the voices' prompts, one after the other, as the current stream makes
        them."""
        self.stream.wait_stream(torch.cuda.current_stream())
        x.record_stream(self.stream)      # its memory is not given out again before it has been read
        with torch.cuda.stream(self.stream):
            q = torch.empty((x.shape[0], self.heads, self.dim), dtype=torch.bfloat16, device="cuda")
            out = torch.empty_like(q)
            self._layers(x, self.voices, q, out, lambda cache: prompt_attention(
                self.device, q, cache, self.voices, out, stream=self.stream.cuda_stream))
            return out

    def step(self):
        """A token for every sequence: `ids` goes in and is replaced by the next."""
        with torch.cuda.stream(self.stream):
            self.kv_lens.add_(1)
            self.positions.add_(1)
            x = self.embed[self.ids]
            x = self._layers(x, self.batch, self.q, self.attended, lambda cache: decode_attention(
                self.device, self.q, cache, self.batch, self.attended, prefix=self.prefix,
                stream=self.stream.cuda_stream), self.positions)
            self.hidden = _rms(x, self.final_norm)
            head_sample(self.device, self.hidden, self.head, self.segment, self.options, stream=self.stream.cuda_stream)

    def capture(self):
        """A graph of one step; a step must have run before, so that every workspace has its size."""
        graph = torch.cuda.CUDAGraph()
        self.stream.synchronize()
        with torch.cuda.graph(graph, stream=self.stream):
            self.step()
        return graph

    def check(self):
        self.device.synchronize(self.stream.cuda_stream)


def main():
    args = argparse.ArgumentParser()
    args.add_argument("--sequences", type=int, default=64)
    args.add_argument("--voice-tokens", type=int, nargs="+", default=[300, 500])
    args.add_argument("--steps", type=int, default=50)
    args = args.parse_args()
    voices = args.voice_tokens
    voice_of = [s * len(voices) // args.sequences for s in range(args.sequences)]
    with Device(0) as device:
        decoder = VoiceDecoder(device, voices, voice_of, args.steps + 1)
        g = torch.Generator().manual_seed(1)
        decoder.read_voices(torch.randn((sum(voices), 1024), generator=g).to(torch.bfloat16).cuda())
        decoder.step()
        graph = decoder.capture()
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        with torch.cuda.stream(decoder.stream):
            start.record()
            for _ in range(args.steps):
                graph.replay()
            end.record()
        decoder.check()
        print(f"{args.sequences} sequences, {len(voices)} voices, {len(decoder.layers)} layers: "
              f"{start.elapsed_time(end) / args.steps * 1e3:.1f} us a step; ids {decoder.ids[:8].tolist()} ...")
        del graph


if __name__ == "__main__":
    main()
