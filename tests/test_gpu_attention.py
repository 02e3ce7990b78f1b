"""Norm, rotation and cache append, prompt attention and decode attention over a paged cache, against plain 64-bit forms
(tests/attention_ref.py, which also derives the bounds)."""

import ctypes

import pytest

from tests import attention_ref as ref

pytestmark = pytest.mark.gpu


class Pool:
    """A cache whose pages are handed out in a shuffled order; every value that no sequence holds is NaN."""

    def __init__(self, n_pages, page, kv, dim, seed, heads_first=False):
        import torch
        from voxwerk_b200 import KvCache
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        shape = (n_pages, kv, page, dim) if heads_first else (n_pages, page, kv, dim)
        self.k, self.v = (torch.full(shape, float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        if heads_first:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.page, self.kv, self.dim = page, kv, dim
        self.free = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.cache = KvCache(self.k, self.v)

    def normal(self, *shape, scale=1.0):
        import torch
        return (torch.randn(shape, generator=self.gen, device="cuda") * scale).to(torch.bfloat16)

    def table(self, lens, fill=True, k_scale=1.3, width=None):
        """Page tables of sequences of these lengths, their keys and values filled in; unused entries name no page."""
        import torch
        counts = [-(-n // self.page) for n in lens]
        t = torch.full((len(lens), max(width or 1, *counts, 1) if counts else 1), -7, dtype=torch.int32)
        for s, (n, c) in enumerate(zip(lens, counts)):
            mine = [self.free.pop() for _ in range(c)]
            t[s, :c] = torch.tensor(mine, dtype=torch.int32)
            if fill and n:
                j = torch.arange(n, device="cuda")
                where = torch.tensor(mine, device="cuda")[j // self.page], j % self.page
                self.k[where] = self.normal(n, self.kv, self.dim, scale=k_scale)
                self.v[where] = self.normal(n, self.kv, self.dim)
        return t.cuda()


def ints(values):
    import torch
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def offsets_of(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


# ---------------------------------------------------------------------------------------------------------- append
ROPE_CASES = [
    # heads, kv, dim, rotary, interleaved, norm, dtype, page, new rows and earlier keys per sequence (None: one row each)
    (16, 8, 128, 128, False, True, "bfloat16", 16, [5, 1, 0, 37], [0, 16, 3, 700]),
    (16, 8, 128, 128, False, True, "float32", 16, None, [0, 15, 16, 300, 31]),
    (4, 2, 64, 64, True, False, "bfloat16", 64, [130, 2], [63, 0]),
    (12, 2, 96, 48, True, True, "float32", 32, [9, 33], [1, 40]),
    (5, 1, 80, 40, False, True, "bfloat16", 128, [17], [128]),
    (6, 3, 80, 80, False, False, "float32", 16, [3, 4, 5, 6], [0, 0, 9, 1]),
    (3, 1, 72, 36, False, True, "bfloat16", 16, [21, 1], [5, 0]),
    (40, 8, 256, 128, False, True, "bfloat16", 256, [3], [255]),
    (2, 2, 248, 30, True, True, "float32", 16, [11], [0]),
    (1, 1, 8, 2, False, True, "bfloat16", 16, [40], [0]),
    (2, 1, 64, 0, False, True, "bfloat16", 16, [7, 9], [0, 2]),
]


def _append(device, heads, kv, dim, rotary, interleaved, norm, dtype, page, new, past, layout="fused", given=False,
            heads_first=False, stream=None, spare=3):
    """One call and its check; the rows past the last offset, the rest of the cache and of q_out keep their values."""
    import torch
    from voxwerk_b200 import KvBatch, RopeTable, rope_append
    seqs = len(past)
    rows = new or [1] * seqs
    total, n = [a + b for a, b in zip(rows, past)], sum(rows) + (spare if new else 0)
    pool = Pool(sum(-(-t // page) for t in total) + 2, page, kv, dim, seed=dim + n, heads_first=heads_first)
    table = pool.table(total, fill=False)
    want_k, want_v = pool.k.clone(), pool.v.clone()
    bound_k = torch.zeros(pool.k.shape, dtype=torch.float64, device="cuda")
    dt = getattr(torch, dtype)
    g = pool.gen
    if layout == "fused":        # one projection's output
        x = (torch.randn((n, (heads + 2 * kv) * dim), generator=g, device="cuda") * 1.5).to(dt)
        q, k, v = (t.view(n, -1, dim) for t in x.split([heads * dim, kv * dim, kv * dim], dim=1))
        q_out = torch.full((n, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    elif layout == "heads_first":
        q, k, v = ((torch.randn((h, n, dim), generator=g, device="cuda") * 1.5).to(dt).transpose(0, 1)
                   for h in (heads, kv, kv))
        q_out = torch.full((heads, n, dim), 7.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    else:                        # nothing aligned beyond its elements
        x = (torch.randn(n * (heads + 2 * kv) * (dim + 1) + 3, generator=g, device="cuda") * 1.5).to(dt)[1:]
        part = lambda at, h: x[at:at + n * h * (dim + 1)].view(n, h, dim + 1)[..., :dim]
        q, k, v = part(0, heads), part(n * heads * (dim + 1), kv), part(n * (heads + kv) * (dim + 1), kv)
        q_out = torch.full((n * heads * (dim + 1) + 1,), 7.0, dtype=torch.bfloat16, device="cuda")[1:].view(
            n, heads, dim + 1)[..., :dim]
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=g, device="cuda")) if norm else None for _ in range(2))
    seq = torch.tensor([s for s, r in enumerate(rows) for _ in range(r)], device="cuda")
    index = torch.tensor([p + i for r, p in zip(rows, past) for i in range(r)], device="cuda")
    positions = None
    place = index
    if given:
        place = (index * 7 + 11) % 900
        positions = torch.full((n,), -5, dtype=torch.int32, device="cuda")
        positions[:place.numel()] = place
    table_rows = int(place.max()) + 1
    rope = RopeTable.build(table_rows, rotary, base=5e5, interleaved=interleaved, linear=2.0) if rotary else None
    batch = KvBatch(table, ints(total), ints(offsets_of(rows)) if new else None)
    rope_append(device, q, k, v, pool.cache, batch, rope, q_out, q_norm=wq, k_norm=wk, eps=1e-5, positions=positions,
                stream=stream)
    torch.cuda.synchronize()
    m = place.numel()
    cos, sin = (rope.cos[place], rope.sin[place]) if rope else (None, None)
    want_q, bound_q = ref.rope(q[:m], wq, 1e-5, cos, sin, interleaved)
    ref.check(q_out[:m], want_q, bound_q, "q_out")
    assert bool((q_out[m:] == 7.0).all()), "rows past the last offset were written"
    new_k, new_bound = ref.rope(k[:m], wk, 1e-5, cos, sin, interleaved)
    where = table.long()[seq, index // page], index % page
    got_k = pool.k[where].clone()
    ref.check(got_k, new_k, new_bound, "keys")
    assert torch.equal(pool.v[where], v[:m].to(torch.bfloat16)), "values are the rounded inputs"
    want_k[where], want_v[where] = got_k, pool.v[where]
    for got, want in ((pool.k, want_k), (pool.v, want_v)):
        assert torch.equal(got.contiguous().view(torch.int16), want.contiguous().view(torch.int16)), \
            "a place of the cache that no row owns was written"


@pytest.mark.parametrize("case", ROPE_CASES, ids=lambda c: f"{c[0]}x{c[2]}r{c[3]}{'i' if c[4] else 'h'}-{c[6]}")
def test_append_matches_formula(device, case):
    _append(device, *case)


@pytest.mark.parametrize("layout", ["heads_first", "loose"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_append_layouts_and_given_positions(device, layout, dtype):
    _append(device, 6, 2, 64, 32, False, True, dtype, 16, [40, 3, 1], [0, 19, 5], layout=layout, given=True)
    _append(device, 6, 2, 64, 64, True, True, dtype, 32, [40, 3, 1], [0, 19, 5], layout=layout, given=True)


def test_append_heads_first_cache_and_many_sequences(device):
    _append(device, 4, 2, 128, 128, False, True, "bfloat16", 16, None, [(37 * i) % 50 for i in range(1500)])
    _append(device, 4, 2, 64, 64, False, True, "bfloat16", 32, [i % 4 for i in range(1100)],
            [(13 * i) % 40 for i in range(1100)], heads_first=True)


def test_append_reports_what_does_not_fit(device):
    """A page outside the cache, a position outside the table and a key index outside the page table are reported; the
    other rows of the call are written."""
    import torch
    from voxwerk_b200 import KvBatch, RopeTable, VwInvalidArgument, VwOutOfRange, rope_append
    pool = Pool(12, 16, 1, 64, seed=1)
    q, k, v = (pool.normal(3, 1, 64) for _ in range(3))
    q_out = torch.zeros_like(q)
    rope = RopeTable.build(64, 64)
    table = pool.table([20, 20, 20], fill=False)
    good = table.clone()
    table[1, 1] = 12
    with pytest.raises(VwOutOfRange, match="page"):
        rope_append(device, q, k, v, pool.cache, KvBatch(table, ints([20, 20, 20])), rope, q_out)
    assert bool(torch.isfinite(pool.k[good.long()[[0, 2], 1], 3]).all())
    assert bool((q_out[1] == 0).all()) and bool((q_out[2] != 0).any())
    with pytest.raises(VwOutOfRange, match="position"):
        rope_append(device, q, k, v, pool.cache, KvBatch(good, ints([20, 20, 20])), rope, q_out, positions=ints([0, 64, 1]))
    with pytest.raises(VwOutOfRange, match="position"):
        rope_append(device, q, k, v, pool.cache, KvBatch(good, ints([20, 20, 20])), rope, q_out, positions=ints([0, -1, 1]))
    with pytest.raises(VwInvalidArgument, match="kv_lens"):
        rope_append(device, q, k, v, pool.cache, KvBatch(good, ints([20, 33, 20])), rope, q_out)
    with pytest.raises(VwInvalidArgument, match="kv_lens"):
        rope_append(device, q, k, v, pool.cache, KvBatch(good, ints([20, 0, 20])), rope, q_out)
    rope_append(device, q, k, v, pool.cache, KvBatch(good, ints([20, 20, 20])), rope, q_out)   # the handle still works


# ------------------------------------------------------------------------------------------------------- attention
def _prompt(device, heads, kv, dim, page, new, past, seed=0, k_scale=1.3, scale=None, heads_first=False, stream=None,
            lse=True, q_layout="rows", width=None, keys=None, check=True):
    """One call and its check.  keys: the key counts, where they are not new + past."""
    import torch
    from voxwerk_b200 import KvBatch, prompt_attention
    total = keys or [a + b for a, b in zip(new, past)]
    pool = Pool(sum(-(-t // page) for t in total) + 2, page, kv, dim, seed=seed, heads_first=heads_first)
    table = pool.table(total, k_scale=k_scale, width=width)
    n = sum(new) + 2
    if q_layout == "rows":
        q = pool.normal(n, heads, dim, scale=1.3)
        out = torch.full((n, heads, dim), 9.0, dtype=torch.bfloat16, device="cuda")
    else:
        q = pool.normal(heads, n + 5, dim + 8, scale=1.3)[:, 2:n + 2, :dim].transpose(0, 1)
        out = torch.full((heads, n, dim), 9.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    ls = torch.full((n, heads), 9.0, device="cuda") if lse else None
    torch.cuda.synchronize()
    prompt_attention(device, q, pool.cache, KvBatch(table, ints(total), ints(offsets_of(new))), out, scale=scale, lse=ls,
                     stream=stream)
    torch.cuda.synchronize()
    if check:
        _check_prompt(pool, table, q, out, ls, new, total, dim ** -0.5 if scale is None else scale)
    return pool, table, q, out, ls


def _check_prompt(pool, table, q, out, ls, new, total, scale):
    import torch
    at = 0
    for s, (r, t) in enumerate(zip(new, total)):
        k, v = (ref.keys_of(c, table[s], t) for c in (pool.k, pool.v))
        for r0 in range(0, r, 512):
            rows = slice(at + r0, at + min(r, r0 + 512))
            limit = t - r + 1 + torch.arange(r0, min(r, r0 + 512), device="cuda")
            want, lse, bound, lse_bound = ref.attend(q[rows], k, v, scale, limit)
            ref.check(out[rows], want, bound, f"sequence {s} rows {rows}")
            if ls is not None:
                ref.check(ls[rows], lse, lse_bound, f"sequence {s} lse")
        at += r
    assert bool((out[at:] == 9.0).all()), "rows past the last offset were written"
    assert ls is None or bool((ls[at:] == 9.0).all())


@pytest.mark.parametrize("heads,kv,dim,page", [(16, 8, 128, 16), (4, 4, 64, 64), (8, 1, 128, 32), (6, 2, 96, 16),
                                               (5, 1, 80, 128), (7, 1, 64, 256), (2, 1, 8, 16), (64, 1, 64, 16),
                                               (3, 3, 120, 32), (20, 4, 128, 128)])
def test_prompt_heads_dims_and_pages(device, heads, kv, dim, page):
    _prompt(device, heads, kv, dim, page, [1, 70, 0, 33, 129], [0, 0, 5, 100, 3], seed=heads)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 511, 640, 1025])
def test_prompt_lengths(device, n):
    _prompt(device, 4, 2, 128, 16, [n], [0], seed=n)
    _prompt(device, 4, 2, 64, 64, [n, 3, n], [77, 0, 128], seed=n)


@pytest.mark.parametrize("past", [1, 127, 128, 500, 4000, 9001])
@pytest.mark.parametrize("new", [1, 5, 64, 200])
def test_prompt_pieces_on_a_long_cache(device, new, past):
    """Few rows over many keys: the work is split over the keys and joined."""
    _prompt(device, 4, 1, 128, 32, [new], [past], seed=new + past)
    _prompt(device, 8, 2, 64, 128, [new, 2], [past, 300], seed=new + past)


def test_prompt_many_sequences_and_long_ones(device):
    _prompt(device, 2, 1, 64, 16, [(7 * i) % 23 for i in range(700)], [(11 * i) % 90 for i in range(700)], seed=3)
    _prompt(device, 4, 2, 128, 64, [3000, 17, 1500, 2], [0, 1200, 900, 2500], seed=4)


def test_prompt_rows_without_keys(device):
    """Sequences with fewer keys than rows: the rows before the first key get 0 and -inf; no keys at all: every row."""
    _prompt(device, 4, 2, 128, 16, [5, 200, 3, 1], None, keys=[3, 60, 0, 0], seed=5)
    _prompt(device, 4, 2, 64, 32, [300], None, keys=[1], seed=6)


def test_prompt_layouts_scale_and_no_lse(device):
    _prompt(device, 6, 2, 64, 16, [40, 130], [0, 9], seed=7, heads_first=True, q_layout="heads_first")
    _prompt(device, 4, 2, 128, 32, [150], [20], seed=8, scale=0.31, lse=False, q_layout="heads_first")
    _prompt(device, 4, 2, 128, 32, [150], [20], seed=8, scale=-0.05)
    _prompt(device, 4, 2, 128, 16, [30, 60], [20, 0], seed=9, width=600)   # a page table far wider than the sequences


def test_prompt_rising_scores(device):
    """Scores whose maximum rises by far more than one exponential's range from tile to tile, and scores in the
    thousands."""
    import torch
    from voxwerk_b200 import KvBatch, prompt_attention
    for order in (1, -1):
        pool = Pool(80, 16, 1, 128, seed=10)
        table = pool.table([1000])
        j = torch.arange(1000, device="cuda")
        where = table.long()[0, j // 16], j % 16
        ramp = torch.linspace(0.02, 6.0, 1000, device="cuda")
        ramp = ramp if order == 1 else ramp.flip(0)
        base = pool.normal(1, 1, 128, scale=1.0).float()
        pool.k[where] = (base * ramp[:, None, None] + 0.02 * pool.normal(1000, 1, 128).float()).to(torch.bfloat16)
        q = (base.repeat(700, 2, 1) * torch.linspace(-4, 4, 700, device="cuda")[:, None, None]).to(torch.bfloat16)
        q = torch.cat([q, q[:2]])
        out = torch.full_like(q, 9.0)
        ls = torch.full((702, 2), 9.0, device="cuda")
        prompt_attention(device, q, pool.cache, KvBatch(table, ints([1000]), ints([0, 700])), out, lse=ls)
        _check_prompt(pool, table, q, out, ls, [700], [1000], 128 ** -0.5)


def test_prompt_keys_that_are_not_finite(device):
    """A key that is not finite, and a value that is not finite of another sequence, reach no row that does not see
    them (the pages' unused places and the pages of no sequence are NaN in every test here)."""
    import torch
    from voxwerk_b200 import KvBatch, prompt_attention
    pool = Pool(60, 16, 2, 64, seed=11)
    new, total = [200, 150, 90], [230, 150, 300]
    table = pool.table(total)
    bad = 170
    pool.k[table.long()[0, bad // 16], bad % 16] = float("nan")
    pool.k[table.long()[2, 250 // 16], 250 % 16] = float("inf")
    pool.v[table.long()[1, :10]] = float("inf")
    q = pool.normal(sum(new), 4, 64)
    out = torch.empty_like(q)
    ls = torch.empty((sum(new), 4), device="cuda")
    prompt_attention(device, q, pool.cache, KvBatch(table, ints(total), ints(offsets_of(new))), out, lse=ls)
    for s, first, count in ((0, 0, bad - 30), (2, 350, 40)):
        k, v = (ref.keys_of(c, table[s], total[s]) for c in (pool.k, pool.v))
        limit = total[s] - new[s] + 1 + torch.arange(count, device="cuda")
        reach = int(limit.max())
        want, lse, bound, lse_bound = ref.attend(q[first:first + count], k[:reach], v[:reach], 64 ** -0.5, limit)
        ref.check(out[first:first + count], want, bound, f"rows before the bad key of sequence {s}")
        ref.check(ls[first:first + count], lse, lse_bound, "lse")
    assert bool(torch.isnan(out[bad - 30:200].float()).all())


def _decode(device, heads, kv, dim, page, lens, prefixes=(), groups=(), seed=0, k_scale=1.3, scale=None,
            heads_first=False, stream=None, extra=0, lse=True):
    """One call and its check.  groups: the first sequence of each prefix's group and past its last (offsets)."""
    import torch
    from voxwerk_b200 import KvBatch, KvPrefix, decode_attention
    pool = Pool(sum(-(-t // page) for t in [*lens, *prefixes]) + 2, page, kv, dim, seed=seed, heads_first=heads_first)
    table, ptable = pool.table(lens, k_scale=k_scale), pool.table(prefixes, k_scale=k_scale) if prefixes else None
    n = len(lens)
    q = pool.normal(n + extra, heads, dim, scale=1.3)
    out = torch.full((n + extra, heads, dim), 9.0, dtype=torch.bfloat16, device="cuda")
    ls = torch.full((n + extra, heads), 9.0, device="cuda") if lse else None
    prefix = KvPrefix(ptable, ints(prefixes), ints(groups)) if prefixes else None
    torch.cuda.synchronize()
    call = lambda: decode_attention(device, q, pool.cache, KvBatch(table, ints(lens)), out, prefix=prefix, scale=scale,
                                    lse=ls, stream=stream)
    call()
    torch.cuda.synchronize()
    check = lambda: _check_decode(pool, table, ptable, q, out, ls, lens, prefixes, groups,
                                  dim ** -0.5 if scale is None else scale)
    check()
    return call, check, out, ls


def _check_decode(pool, table, ptable, q, out, ls, lens, prefixes, groups, scale):
    import torch
    shared = [tuple(ref.keys_of(c, ptable[g], p) for c in (pool.k, pool.v)) for g, p in enumerate(prefixes)]
    for s, t in enumerate(lens):
        k, v = (ref.keys_of(c, table[s], t) for c in (pool.k, pool.v))
        for g in range(len(prefixes)):
            if groups[g] <= s < groups[g + 1]:
                k, v = torch.cat([shared[g][0], k]), torch.cat([shared[g][1], v])
        want, lse, bound, lse_bound = ref.attend(q[s:s + 1], k, v, scale)
        ref.check(out[s:s + 1], want, bound, f"sequence {s} ({t} keys)")
        if ls is not None:
            ref.check(ls[s:s + 1], lse, lse_bound, f"sequence {s} lse")
    assert bool((out[len(lens):] == 9.0).all())


@pytest.mark.parametrize("heads,kv,dim,page", [(16, 8, 128, 16), (4, 4, 64, 64), (8, 1, 128, 32), (6, 2, 96, 16),
                                               (5, 1, 80, 128), (7, 1, 64, 256), (2, 1, 8, 16), (64, 1, 64, 16),
                                               (34, 2, 128, 64), (3, 3, 120, 32)])
def test_decode_heads_dims_and_pages(device, heads, kv, dim, page):
    _decode(device, heads, kv, dim, page, [1, 0, 70, 33, 129, 400], seed=heads)
    _decode(device, heads, kv, dim, page, [1, 0, 70, 33, 129, 400], [300, 17], [0, 4, 6], seed=heads + 1)


@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 63, 64, 65, 128, 129, 700, 5000, 33001])
def test_decode_one_sequence(device, n):
    _decode(device, 4, 2, 128, 16, [n], seed=n)
    _decode(device, 8, 1, 64, 64, [n], [n], [0, 1], seed=n)


@pytest.mark.parametrize("n,prefix", [(2, 90), (9, 4099), (40, 1), (64, 640), (130, 129), (300, 2000), (65, 16001)])
def test_decode_one_prefix(device, n, prefix):
    lens = [(37 * i) % 150 for i in range(n)]
    _decode(device, 4, 2, 128, 32, lens, [prefix], [0, n], seed=n, extra=1)


def test_decode_groups(device):
    lens = [(29 * i) % 200 for i in range(120)]
    # uneven groups, one of no sequence, one without keys, sequences before the first and after the last group
    _decode(device, 8, 2, 64, 16, lens, [400, 0, 77, 1300], [3, 50, 60, 60, 110], seed=1)
    _decode(device, 6, 2, 128, 16, lens, [0, 0], [0, 60, 120], seed=2)
    _decode(device, 6, 2, 128, 16, [0] * 20, [130, 0, 64], [0, 8, 12, 20], seed=3)     # prefixes alone, and nothing
    _decode(device, 2, 1, 64, 16, lens, [20 + i for i in range(40)], list(range(0, 123, 3)), seed=4)   # 40 groups of 3


def test_decode_layouts_scale_and_rising_scores(device):
    _decode(device, 6, 2, 64, 16, [300, 20, 0], [100], [0, 2], seed=5, heads_first=True, scale=0.4)
    _decode(device, 4, 2, 128, 64, [1500, 800], [900], [0, 2], seed=6, k_scale=25.0, lse=False)


def test_attention_repeats_and_streams(device):
    """The same call gives the same bits, on the handle's stream, on a caller's, and on two in turn (the library orders
    its workspace between them)."""
    import torch
    lens = [(53 * i) % 900 for i in range(30)]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    calls = [_decode(device, 8, 2, 128, 16, lens, [3000], [0, 30], seed=7 + i, stream=s.cuda_stream)
             for i, s in enumerate((a, b))]
    want = [(o.clone(), l.clone()) for _, _, o, l in calls]
    for _ in range(20):
        for call, _, o, l in calls:
            o.record_stream(a), l.record_stream(b)
            call()
    torch.cuda.synchronize()
    device.synchronize(a.cuda_stream)
    for (call, check, o, l), (wo, wl) in zip(calls, want):
        assert torch.equal(o.view(torch.int16), wo.view(torch.int16)) and torch.equal(l, wl)
        check()
    for new, past in (([700, 40], [0, 3000]), ([3], [7000])):
        outs = [_prompt(device, 4, 2, 128, 16, new, past, seed=12, stream=s)[3:] for s in (None, a.cuda_stream, None)]
        for o, l in outs[1:]:
            assert torch.equal(o.view(torch.int16), outs[0][0].view(torch.int16)) and torch.equal(l, outs[0][1])


def test_step_in_a_cuda_graph(device):
    """A decode step (append, then attention) captured once and replayed as the sequences grow."""
    import torch
    from voxwerk_b200 import KvBatch, KvPrefix, RopeTable, decode_attention, rope_append
    pool = Pool(200, 16, 2, 128, seed=13)
    lens = [30, 0, 17, 63]
    table, ptable = pool.table([n + 5 for n in lens], fill=False), pool.table([500])
    for s, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        where = table[s].long()[j // 16], j % 16
        pool.k[where], pool.v[where] = pool.normal(n, 2, 128), pool.normal(n, 2, 128)
    kv_lens = ints(lens)
    batch, prefix = KvBatch(table, kv_lens), KvPrefix(ptable, ints([500]), ints([0, 3]))
    rope = RopeTable.build(1000, 128)
    qkv = pool.normal(4, 8 * 128)
    q, k, v = qkv[:, :512].view(4, 4, 128), qkv[:, 512:768].view(4, 2, 128), qkv[:, 768:].view(4, 2, 128)
    q_out, out = (torch.empty((4, 4, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    stream = torch.cuda.Stream()

    def step():
        kv_lens.add_(1)
        rope_append(device, q, k, v, pool.cache, batch, rope, q_out, stream=stream.cuda_stream)
        decode_attention(device, q_out, pool.cache, batch, out, prefix=prefix, stream=stream.cuda_stream)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for i in range(2, 5):
        qkv.copy_(pool.normal(4, 8 * 128))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        device.synchronize(stream.cuda_stream)
        now = [n + i for n in lens]
        assert kv_lens.tolist() == now
        full = out.new_full((4, 4, 128), 9.0)
        full.copy_(out)
        _check_decode(pool, table, ptable, q_out, full, None, now, [500], [0, 3], 128 ** -0.5)


def test_attention_past_32_bit_offsets(device):
    """Pages more than 2^31 elements into the cache."""
    import torch
    from voxwerk_b200 import KvBatch, KvCache, KvPrefix, decode_attention, prompt_attention, rope_append
    pages = 2 ** 31 // (64 * 8 * 128) + 40
    k, v = (torch.empty((pages, 64, 8, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = KvCache(k, v)
    table = (pages - 1 - torch.arange(6, dtype=torch.int32, device="cuda")).view(2, 3)
    g = torch.Generator(device="cuda").manual_seed(3)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
    new_k, new_v, q = normal(300, 8, 128), normal(300, 8, 128), normal(300, 16, 128)
    q_out = torch.empty_like(q)
    batch = KvBatch(table, ints([150, 150]), ints([0, 150, 300]))
    rope_append(device, q, new_k, new_v, cache, batch, None, q_out)
    assert torch.equal(q_out, q)
    out = torch.empty_like(q)
    prompt_attention(device, q, cache, batch, out)
    for s in range(2):
        rows = slice(150 * s, 150 * s + 150)
        want, _, bound, _ = ref.attend(q[rows], new_k[rows].double(), new_v[rows].double(), 128 ** -0.5,
                                       1 + torch.arange(150, device="cuda"))
        ref.check(out[rows], want, bound, f"sequence {s}")
    two = torch.empty_like(q[:2])
    decode_attention(device, q[:2], cache, KvBatch(table, ints([150, 150])), two,
                     prefix=KvPrefix(table[:1], ints([150]), ints([0, 2])))
    both = lambda x, s: torch.cat([x[:150], x[150 * s:150 * s + 150]]).double()
    for s in range(2):
        want, _, bound, _ = ref.attend(q[s:s + 1], both(new_k, s), both(new_v, s), 128 ** -0.5)
        ref.check(two[s:s + 1], want, bound, f"decode {s}")


def test_attention_reports_what_does_not_fit(device):
    """Pages outside the cache, key counts past the page table, and offsets that do not ascend are reported, not
    followed; the next call is right."""
    import torch
    from voxwerk_b200 import KvBatch, KvPrefix, VwInvalidArgument, VwOutOfRange, decode_attention, prompt_attention
    pool = Pool(40, 16, 2, 64, seed=14)
    table, ptable = pool.table([100, 60]), pool.table([50])
    q = pool.normal(20, 4, 64)
    out = torch.empty_like(q)
    bad = table.clone()
    bad[0, 2] = 40
    with pytest.raises(VwOutOfRange, match="page"):
        prompt_attention(device, q, pool.cache, KvBatch(bad, ints([100, 60]), ints([0, 10, 20])), out)
    with pytest.raises(VwOutOfRange, match="page"):
        decode_attention(device, q, pool.cache, KvBatch(bad, ints([100, 60])), out)
    bad[0, 2] = -1
    with pytest.raises(VwOutOfRange, match="page"):
        decode_attention(device, q, pool.cache, KvBatch(table, ints([100, 60])), out,
                         prefix=KvPrefix(bad[:1], ints([50]), ints([0, 2])))
    for lens in ([100, 113], [-1, 60]):
        with pytest.raises(VwInvalidArgument, match="kv_lens"):
            prompt_attention(device, q, pool.cache, KvBatch(table, ints(lens), ints([0, 10, 20])), out)
        with pytest.raises(VwInvalidArgument, match="kv_lens"):
            decode_attention(device, q, pool.cache, KvBatch(table, ints(lens)), out)
    for offsets in ([0, 15, 10], [0, 10, 21], [-3, 10, 20]):
        with pytest.raises(VwInvalidArgument, match="q_offsets"):
            prompt_attention(device, q, pool.cache, KvBatch(table, ints([100, 60]), ints(offsets)), out)
    for groups in ([2, 0], [0, 3], [-1, 2]):
        with pytest.raises(VwInvalidArgument, match="group_offsets"):
            decode_attention(device, q, pool.cache, KvBatch(table, ints([100, 60])), out,
                             prefix=KvPrefix(ptable, ints([50]), ints(groups)))
    with pytest.raises(VwInvalidArgument, match="kv_lens"):
        decode_attention(device, q, pool.cache, KvBatch(table, ints([100, 60])), out,
                         prefix=KvPrefix(ptable, ints([65]), ints([0, 2])))
    out.fill_(9.0)
    ls = torch.full((20, 4), 9.0, device="cuda")
    prompt_attention(device, q, pool.cache, KvBatch(table, ints([100, 60]), ints([0, 10, 18])), out, lse=ls)
    _check_prompt(pool, table, q, out, ls, [10, 8], [100, 60], 0.125)
    out.fill_(9.0)
    decode_attention(device, q, pool.cache, KvBatch(table, ints([100, 60])), out,
                     prefix=KvPrefix(ptable, ints([50]), ints([0, 2])))
    _check_decode(pool, table, ptable, q, out, None, [100, 60], [50], [0, 2], 0.125)


def test_refused_arguments(device):
    """Sizes, strides, types and pointers that the operators do not take raise before anything runs."""
    import torch
    from voxwerk_b200 import (KvBatch, KvCache, RopeTable, VwInvalidArgument, decode_attention, prompt_attention,
                              rope_append)
    from voxwerk_b200._lib import VwKvCache
    pool = Pool(8, 16, 2, 64, seed=15)
    table = pool.table([20, 20])
    batch = KvBatch(table, ints([20, 20]), ints([0, 1, 2]))
    q = pool.normal(2, 4, 64)
    out = torch.empty_like(q)
    good = lambda call, **kw: call(device, q, pool.cache, batch, out, **kw)
    for call in (prompt_attention, decode_attention):
        good(call)
        with pytest.raises(TypeError):
            call(device, q.float(), pool.cache, batch, out)
        with pytest.raises(TypeError):
            call(device, q.cpu(), pool.cache, batch, out)
        with pytest.raises(ValueError):
            call(device, q[..., :32], pool.cache, batch, out)
        with pytest.raises(ValueError):
            call(device, q, pool.cache, batch, out[:1])
        with pytest.raises(ValueError):
            good(call, lse=torch.empty((2, 5), device="cuda"))
        with pytest.raises(VwInvalidArgument, match="n_q_heads"):
            call(device, q[:, :3], pool.cache, batch, out[:, :3])
        with pytest.raises(VwInvalidArgument, match="scale"):
            good(call, scale=float("nan"))
        flat = torch.empty(2 * 4 * 64 + 8, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(VwInvalidArgument, match="aligned"):
            call(device, flat[1:513].view(2, 4, 64), pool.cache, batch, out)
        loose = torch.empty((2, 4, 68), dtype=torch.bfloat16, device="cuda")[..., :64]
        with pytest.raises(VwInvalidArgument, match="strides"):
            call(device, loose, pool.cache, batch, out)
        wide = Pool(8, 16, 2, 136, seed=16)
        with pytest.raises(VwInvalidArgument, match="head_dim"):
            call(device, wide.normal(2, 4, 136), wide.cache, batch, wide.normal(2, 4, 136))
        with pytest.raises(VwInvalidArgument, match="page_size"):
            call(device, q, KvCache.empty(4, 24, 2, 64), batch, out)
    with pytest.raises(VwInvalidArgument, match="n_rows"):
        prompt_attention(device, pool.normal(3, 4, 64), pool.cache, KvBatch(table, ints([20, 20])), pool.normal(3, 4, 64))
    with pytest.raises(VwInvalidArgument, match="n_rows"):
        decode_attention(device, q[:1], pool.cache, batch, out[:1])
    rope = RopeTable.build(32, 64)
    k = pool.normal(2, 2, 64)
    rope_append(device, q, k, k, pool.cache, batch, rope, out)
    with pytest.raises(TypeError):
        rope_append(device, q.half(), k.half(), k.half(), pool.cache, batch, rope, out)
    with pytest.raises(TypeError):
        rope_append(device, q, k.float(), k, pool.cache, batch, rope, out)
    with pytest.raises(ValueError):
        rope_append(device, q, k[:1], k, pool.cache, batch, rope, out)
    with pytest.raises(VwInvalidArgument, match="rotary_dim"):
        rope_append(device, q, k, k, pool.cache, batch, RopeTable.build(32, 66), out)
    with pytest.raises(VwInvalidArgument, match="eps"):
        rope_append(device, q, k, k, pool.cache, batch, rope, out, eps=-1.0)
    with pytest.raises(ValueError):
        KvCache(pool.k, pool.v[:4])
    with pytest.raises(TypeError):
        KvBatch(table.long(), ints([20, 20]))
    assert ctypes.sizeof(VwKvCache) == 56
    for call in (prompt_attention, decode_attention):   # no sequences, no rows: nothing to do
        call(device, q[:0], pool.cache, KvBatch(table[:0], ints([])), out[:0])
