"""The attention operators around a decoder step, as cases to time and compare.

Three operators share one paged key/value cache ([n_pages, page_size, n_kv_heads, head_dim] bf16 each for keys and
values; a sequence's page table lists its pages in order):

* ``append``: each query and key head normalised (RMS) and rotated to its position, keys and values written into the
  cache, queries written out;
* ``prompt``: causal attention of packed sequences of different lengths, whose keys are in the cache;
* ``decode``: one new token per sequence, groups of sequences sharing a prefix that the cache holds once.

``run`` computes them in plain torch operations (``own`` false) or through voxwerk_b200 (``own`` true).  ``exact``
computes the same outputs in 64 bits from the definitions, one sequence and head group at a time.
"""

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
_session = {}


# ------------------------------------------------------------------------------------------------------------- cases
def _case(op, name=None, **kw):
    c = {"op": op, **kw}
    if name is not None:
        c["name"] = name
    return c


def _append(name=None, *, seqs, lo, hi, past=0, heads=16, kv_heads=8, dim=128, rotary=128, interleaved=False, norm=True,
            dtype="bfloat16", scaling=1.0, page=16):
    return _case("append", name, seqs=seqs, lo=lo, hi=hi, past=past, heads=heads, kv_heads=kv_heads, dim=dim,
                 rotary=rotary, interleaved=interleaved, norm=norm, dtype=dtype, scaling=scaling, page=page)


def _prompt(name=None, *, seqs, lo, hi, past=0, heads=16, kv_heads=8, dim=128, page=16):
    return _case("prompt", name, seqs=seqs, lo=lo, hi=hi, past=past, heads=heads, kv_heads=kv_heads, dim=dim, page=page)


def _decode(name=None, *, seqs, lo, hi, groups=0, prefix_lo=0, prefix_hi=0, heads=16, kv_heads=8, dim=128, page=16):
    return _case("decode", name, seqs=seqs, lo=lo, hi=hi, groups=groups, prefix_lo=prefix_lo, prefix_hi=prefix_hi,
                 heads=heads, kv_heads=kv_heads, dim=dim, page=page)


def listed():
    return [
        # one job's next token: the smallest call of a generation loop
        _append("append one token", seqs=1, lo=1, hi=1, past=350),
        # one frame of a full batch, from projections that come out in fp32
        _append("append a frame of 64 fp32", seqs=64, lo=1, hi=1, past=600, dtype="float32"),
        # interleaved pairs over half of each head, positions scaled for a context longer than trained on, no norm
        _append("append scaled interleaved", seqs=5, lo=90, hi=900, past=4000, heads=12, kv_heads=2, dim=96, rotary=48,
                interleaved=True, norm=False, scaling=4.0, page=64),
        # the prompts of a whole batch at once
        _append("append a batch of prompts", seqs=24, lo=150, hi=1700, page=32),
        # one short text prompt
        _prompt("prompt of 37", seqs=1, lo=37, hi=37),
        # voice-clone prompts of a batch, packed
        _prompt("prompts packed", seqs=12, lo=170, hi=1300),
        # a long document in one piece
        _prompt("prompt of 7937", seqs=1, lo=7937, hi=7937, page=64),
        # the next pieces of two long prompts, most of whose keys are cached already
        _prompt("prompt pieces on a long cache", seqs=2, lo=130, hi=250, past=9001, heads=32, kv_heads=4, dim=64,
                page=128),
        # one job alone, no shared prefix
        _decode("decode one", seqs=1, lo=700, hi=700),
        # a frame of 64 jobs that speak with one voice
        _decode("decode 64 on one voice", seqs=64, lo=20, hi=600, groups=1, prefix_lo=4099, prefix_hi=4099),
        # four voices, narrow heads, eight query heads to a key head
        _decode("decode 50 on four voices", seqs=50, lo=60, hi=900, groups=4, prefix_lo=250, prefix_hi=3000, heads=32,
                kv_heads=4, dim=64, page=64),
        # a full server: long prefix, long generations
        _decode("decode 256 on a long prefix", seqs=256, lo=100, hi=2000, groups=1, prefix_lo=16001, prefix_hi=16001,
                page=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _shape(rng):
    kv = rng.choice([1, 2, 4, 8])
    return dict(heads=kv * rng.choice([1, 2, 2, 3, 4, 5, 8]), kv_heads=kv, dim=rng.choice([64, 64, 80, 96, 128, 128]),
                page=rng.choice([16, 32, 64, 128]))


def draw(rng):
    op = rng.choice(["append", "prompt", "decode"])
    shape = _shape(rng)
    if op == "append":
        dim = shape["dim"]
        if rng.random() < 0.5:   # a step of a batch
            seqs = _log(rng, 1, 512)
            lo = hi = 1
            past = _log(rng, 1, 900)
        else:                    # prompts
            seqs = _log(rng, 1, 24)
            hi = _log(rng, 2, 1700)
            lo = rng.randint(1, hi)
            past = rng.choice([0, _log(rng, 1, 4000)])
        return _append(seqs=seqs, lo=lo, hi=hi, past=past, rotary=rng.choice([dim, dim, dim // 2]),
                       interleaved=rng.random() < 0.4, norm=rng.random() < 0.7,
                       dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), scaling=rng.choice([1.0, 1.0, 2.5, 8.0]),
                       **shape)
    if op == "prompt":
        while True:
            seqs, hi = _log(rng, 1, 16), _log(rng, 1, 6000)
            lo = rng.randint(max(1, hi // 8), hi)
            past = rng.choice([0, 0, _log(rng, 1, 8000)])
            case = _prompt(seqs=seqs, lo=lo, hi=hi, past=past, **shape)
            if seqs * shape["heads"] * hi * (past + hi) <= 5e8 and work(case)["flops"] <= 2.4e11:
                return case
    while True:
        seqs, hi = _log(rng, 1, 256), _log(rng, 2, 2000)
        lo = rng.randint(1, hi)
        groups = rng.choice([0, 1, 1, 1, 2, 4])
        phi = _log(rng, 16, 16000)
        plo = rng.randint(1, phi)
        if groups > seqs:
            continue
        case = _decode(seqs=seqs, lo=lo, hi=hi, groups=groups, prefix_lo=plo if groups else 0,
                       prefix_hi=phi if groups else 0, **shape)
        if work(case)["bytes"] <= 1e9 and seqs * shape["heads"] * (groups * phi + hi) <= 3e8:
            return case


def _lengths(n, lo, hi):
    """n lengths from lo to hi, spread over the logarithm, in no order."""
    if lo == hi:
        return [lo] * n
    return [min(hi, max(lo, round(lo * (hi / lo) ** ((0.5 + 0.6180339887 * i) % 1.0)))) for i in range(n)]


def _group_sizes(case):
    """Sequences of each group: uneven, every group at least one."""
    n, g = case["seqs"], case["groups"]
    cuts = [round(n * (i / g) ** 1.3) for i in range(g + 1)] if g else [0]
    for i in range(1, g + 1):
        cuts[i] = max(cuts[i], cuts[i - 1] + 1)
    for i in range(g, 0, -1):
        cuts[i] = min(cuts[i], n - (g - i))
    return [b - a for a, b in zip(cuts, cuts[1:])]


def work(case):
    lens = _lengths(case["seqs"], case["lo"], case["hi"])
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        rows, size = sum(lens), 4 if case["dtype"] == "float32" else 2
        positions = max(lens)   # every sequence starts at `past`: the longest one's rows of the table
        return {"bytes": rows * (h + 2 * kv) * d * (size + 2) + positions * case["rotary"] * 4 + rows * 8,
                "flops": rows * (h + kv) * (3 * case["rotary"] + (4 * d if case["norm"] else 0))}
    if case["op"] == "prompt":
        rows = sum(lens)
        pairs = sum(n * case["past"] + n * (n + 1) // 2 for n in lens)
        keys = sum(n + case["past"] for n in lens)
        return {"bytes": 4 * rows * h * d + 4 * keys * kv * d + 4 * rows * h, "flops": 4 * pairs * h * d}
    prefixes = _lengths(case["groups"], case["prefix_lo"], case["prefix_hi"])
    shared = sum(n * p for n, p in zip(_group_sizes(case), prefixes))
    return {"bytes": 4 * case["seqs"] * h * d + 4 * (sum(lens) + sum(prefixes)) * kv * d + 4 * case["seqs"] * h,
            "flops": 4 * (sum(lens) + shared) * h * d}


# ------------------------------------------------------------------------------------------------------------ inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _page_tables(counts, first_free, order, width):
    """Page tables of sequences with `counts` pages each, taken from the shuffled pool `order`."""
    table = torch.zeros((len(counts), max(width, 1)), dtype=torch.int32)
    at = first_free
    for row, n in enumerate(counts):
        table[row, :n] = order[at:at + n]
        at += n
    return table.to(DEVICE), at


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    lens = _lengths(case["seqs"], case["lo"], case["hi"])
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(dtype)

    totals = lens if case["op"] == "decode" else [n + case["past"] for n in lens]
    prefixes = _lengths(case["groups"], case["prefix_lo"], case["prefix_hi"]) if case["op"] == "decode" else []
    counts = [-(-n // page) for n in totals]
    prefix_counts = [-(-n // page) for n in prefixes]
    n_pages = sum(counts) + sum(prefix_counts) + 3
    order = torch.randperm(n_pages, generator=cpu).to(torch.int32)
    table, used = _page_tables(counts, 0, order, max(counts))
    s = {"case": dict(case), "seqs": case["seqs"], "max_keys": max(totals), "max_rows": max(lens), "table": table,
         "kv_lens": _ints(totals),
         "k_cache": normal(n_pages, page, kv, d, scale=1.3), "v_cache": normal(n_pages, page, kv, d)}
    if case["op"] != "decode":
        offsets = [0]
        for n in lens:
            offsets.append(offsets[-1] + n)
        s["offsets"] = _ints(offsets)
        rows = offsets[-1]
    if case["op"] == "append":
        dtype = getattr(torch, case["dtype"])
        s["qkv"] = normal(rows, (h + 2 * kv) * d, scale=1.5, dtype=dtype)   # a fused projection's output
        s["q_norm"] = 1 + 0.2 * normal(d, dtype=torch.float32) if case["norm"] else None
        s["k_norm"] = 1 + 0.2 * normal(d, dtype=torch.float32) if case["norm"] else None
        angles = _angles(torch.arange(max(totals), dtype=torch.float64, device=DEVICE), case)
        s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()     # a table, laid out once
        s["q_out"] = torch.empty((rows, h, d), dtype=torch.bfloat16, device=DEVICE)
    else:
        rows = case["seqs"] if case["op"] == "decode" else rows
        s["q"] = normal(rows, h, d, scale=1.3)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((rows, h), dtype=torch.float32, device=DEVICE)
    if prefixes:
        s["prefix_table"], _ = _page_tables(prefix_counts, used, order, max(prefix_counts))
        s["prefix_lens"] = _ints(prefixes)
        s["max_prefix"] = max(prefixes)
        sizes = _group_sizes(case)
        s["group_offsets"] = _ints([sum(sizes[:i]) for i in range(len(sizes) + 1)])
    if own:
        s["handles"] = _handles(s)
    return s


def _angles(positions, case):
    """Rotation angles [positions, rotary / 2] in 64 bits: base 1e6, positions divided by the scaling factor."""
    half = case["rotary"] // 2
    freq = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=positions.device) / half)
    return (positions / case["scaling"])[:, None] * freq


def _handles(s):
    """What a program of the framework keeps across calls: the device handle, and the cache, batch, prefix and table
    it describes once."""
    import voxwerk_b200 as vw
    if not _session:
        _session.update(device=vw.Device(0), stream=torch.cuda.Stream())
    a = {"vw": vw, "device": _session["device"], "stream": _session["stream"].cuda_stream,
         "cache": vw.KvCache(s["k_cache"], s["v_cache"]), "prefix": None,
         "batch": vw.KvBatch(s["table"], s["kv_lens"], s.get("offsets"))}
    if "group_offsets" in s:
        a["prefix"] = vw.KvPrefix(s["prefix_table"], s["prefix_lens"], s["group_offsets"])
    if "cos" in s:
        a["rope"] = vw.RopeTable(s["cos"], s["sin"], interleaved=s["case"]["interleaved"])
    return a


# ------------------------------------------------------------------------------------------------------------ passes
def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _split_qkv(s):
    c = s["case"]
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    rows = s["qkv"].shape[0]
    q, k, v = s["qkv"].split([h * d, kv * d, kv * d], dim=1)
    return q.view(rows, h, d), k.view(rows, kv, d), v.view(rows, kv, d)


def _own_append(s):
    a = s["handles"]
    q, k, v = _split_qkv(s)
    a["vw"].rope_append(a["device"], q, k, v, a["cache"], a["batch"], a["rope"], s["q_out"], q_norm=s["q_norm"],
                        k_norm=s["k_norm"], eps=EPS, stream=a["stream"])
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_prompt(s):
    a = s["handles"]
    a["vw"].prompt_attention(a["device"], s["q"], a["cache"], a["batch"], s["out"], lse=s["lse"], stream=a["stream"])
    return {"out": s["out"], "lse": s["lse"]}


def _own_decode(s):
    a = s["handles"]
    a["vw"].decode_attention(a["device"], s["q"], a["cache"], a["batch"], s["out"], prefix=a["prefix"], lse=s["lse"],
                             stream=a["stream"])
    return {"out": s["out"], "lse": s["lse"]}


def _row_places(s, rows):
    """Sequence and place among its keys of each packed row."""
    row = torch.arange(rows, device=DEVICE)
    seq = torch.searchsorted(s["offsets"][1:].long(), row, right=True)
    place = s["kv_lens"].long()[seq] - s["offsets"].long()[seq + 1] + row
    return seq, place


def _plain_append(s):
    c = s["case"]
    q, k, v = (x.float() for x in _split_qkv(s))
    seq, place = _row_places(s, q.shape[0])
    cos, sin = s["cos"][place][:, None], s["sin"][place][:, None]
    half = c["rotary"] // 2
    even = torch.arange(half, device=DEVICE) * 2 if c["interleaved"] else torch.arange(half, device=DEVICE)
    odd = even + 1 if c["interleaved"] else even + half

    def turned(x, weight):
        if weight is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
        y = x.clone()
        y[..., even] = x[..., even] * cos - x[..., odd] * sin
        y[..., odd] = x[..., odd] * cos + x[..., even] * sin
        return y

    page = c["page"]
    s["q_out"].copy_(turned(q, s["q_norm"]))
    slot = s["table"].long()[seq, place // page], place % page
    s["k_cache"][slot] = turned(k, s["k_norm"]).bfloat16()
    s["v_cache"][slot] = v.bfloat16()
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _gathered(cache, table, keys, page):
    """[n, heads, keys, dim] in 32 bits: the first `keys` rows of each sequence of a page table."""
    j = torch.arange(keys, device=DEVICE)
    return cache[table.long()[:, j // page], j % page].float().transpose(1, 2)


def _attend(scores, values):
    """softmax(scores) @ values and log sum exp; rows whose scores are all -inf give zeros and -inf."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ values) / torch.where(total == 0, torch.ones_like(total), total)
    return out, (top + torch.log(total))[..., 0]


def _plain_prompt(s):
    c = s["case"]
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    n, rows, keys = s["seqs"], s["max_rows"], s["max_keys"]
    seq, place = _row_places(s, s["q"].shape[0])
    first = (s["kv_lens"] - (s["offsets"][1:] - s["offsets"][:-1])).long()
    q = torch.zeros((n, rows, h, d), device=DEVICE)
    q[seq, place - first[seq]] = s["q"].float()
    q = q.view(n, rows, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)
    k, v = (_gathered(x, s["table"], keys, c["page"]) for x in (s["k_cache"], s["v_cache"]))
    scores = (q @ k.transpose(-1, -2)) * d ** -0.5
    at = first[:, None] + torch.arange(rows, device=DEVICE)
    seen = torch.arange(keys, device=DEVICE) <= at[..., None]
    scores = scores.view(n, kv, h // kv, rows, keys)
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    out, lse = _attend(scores.view(n, kv, -1, keys), v)
    out = out.view(n, kv, h // kv, rows, d).permute(0, 3, 1, 2, 4).reshape(n, rows, h, d)
    lse = lse.view(n, h, rows).transpose(1, 2)
    mine = seq, place - first[seq]
    s["out"].copy_(out[mine])
    s["lse"].copy_(lse[mine])
    return {"out": s["out"], "lse": s["lse"]}


def _plain_decode(s):
    c = s["case"]
    h, kv, d, page, n, keys = c["heads"], c["kv_heads"], c["dim"], c["page"], s["seqs"], s["max_keys"]
    q = s["q"].float().view(n, kv, h // kv, d)
    k, v = (_gathered(x, s["table"], keys, page) for x in (s["k_cache"], s["v_cache"]))
    seen = torch.arange(keys, device=DEVICE) < s["kv_lens"][:, None]
    scores = (q @ k.transpose(-1, -2)).masked_fill(~seen[:, None, None], float("-inf")) * d ** -0.5
    if "group_offsets" not in s:
        out, lse = _attend(scores, v)
    else:
        p = s["max_prefix"]
        groups = c["groups"]
        pk, pv = (_gathered(x, s["prefix_table"], p, page) for x in (s["k_cache"], s["v_cache"]))
        # every sequence against every group's prefix; the other groups' are masked
        pk, pv = (x.permute(1, 0, 2, 3).reshape(kv, groups * p, d) for x in (pk, pv))
        rows = q.transpose(0, 1).reshape(kv, -1, d)
        shared = (rows @ pk.transpose(-1, -2)).view(kv, n, h // kv, groups * p).transpose(0, 1) * d ** -0.5
        group = torch.searchsorted(s["group_offsets"][1:].long(), torch.arange(n, device=DEVICE), right=True)
        j = torch.arange(groups * p, device=DEVICE)
        visible = (j // p == group[:, None]) & (j % p < s["prefix_lens"].long()[group][:, None])
        shared = shared.masked_fill(~visible[:, None, None], float("-inf"))
        top = torch.maximum(shared.amax(-1, keepdim=True), scores.amax(-1, keepdim=True))
        e, f = torch.exp(shared - top), torch.exp(scores - top)
        total = e.sum(-1, keepdim=True) + f.sum(-1, keepdim=True)
        first = (e.transpose(0, 1).reshape(kv, -1, groups * p) @ pv).view(kv, n, h // kv, d).transpose(0, 1)
        out, lse = (first + f @ v) / total, (top + torch.log(total))[..., 0]
    s["out"].copy_(out.reshape(n, h, d))
    s["lse"].copy_(lse.reshape(n, h))
    return {"out": s["out"], "lse": s["lse"]}


_OWN = {"append": _own_append, "prompt": _own_prompt, "decode": _own_decode}
_PLAIN = {"append": _plain_append, "prompt": _plain_prompt, "decode": _plain_decode}


# ----------------------------------------------------------------------------------------------------- 64-bit values
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "prompt": _exact_prompt, "decode": _exact_decode}[case["op"]](s, case)


def _rows_of(cache, table_row, count, page):
    """The first `count` rows of one sequence, [count, heads, dim], in 64 bits."""
    pages = table_row[: -(-count // page)].long()
    return cache[pages].flatten(0, 1)[:count].double()


def _softmax_of(q, k, v, limit=None):
    """One sequence's rows q [h, r, d] over keys [kv, n, d]; row i sees the first limit[i] keys (all where None)."""
    h, r, d = q.shape
    out = torch.empty_like(q)
    lse = torch.empty((h, r), dtype=torch.float64, device=DEVICE)
    each = h // k.shape[0]
    for head in range(h):
        z = q[head] @ k[head // each].T / math.sqrt(d)
        if limit is not None:
            z[torch.arange(k.shape[1], device=DEVICE)[None, :] >= limit[:, None]] = -math.inf
        lse[head] = torch.logsumexp(z, dim=1)
        out[head] = torch.exp(z - lse[head][:, None]) @ v[head // each]
    return out, lse


def _exact_append(s, case):
    h, kv, d, page, half = case["heads"], case["kv_heads"], case["dim"], case["page"], case["rotary"] // 2
    x = s["qkv"].double().view(-1, h + 2 * kv, d)
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    lens = _lengths(case["seqs"], case["lo"], case["hi"])
    place = torch.cat([torch.arange(n, device=DEVICE) for n in lens]) + case["past"]
    if case["norm"]:
        weight = torch.cat([s["q_norm"].double().expand(h, d), s["k_norm"].double().expand(kv, d)])
        scale = torch.rsqrt(x[:, :h + kv].pow(2).mean(2) + EPS)
        x = torch.cat([x[:, :h + kv] * scale[..., None] * weight, x[:, h + kv:]], dim=1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE), _angles(place.double(), case))[:, None]
    head = x[:, :h + kv, :2 * half]
    if case["interleaved"]:
        z = torch.complex(head[..., 0::2], head[..., 1::2]) * turn
        head = torch.stack([z.real, z.imag], dim=-1).flatten(2)
    else:
        z = torch.complex(head[..., :half], head[..., half:]) * turn
        head = torch.cat([z.real, z.imag], dim=-1)
    turned = torch.cat([head, x[:, :h + kv, 2 * half:]], dim=2)
    at = 0
    for i, n in enumerate(lens):
        p = torch.arange(case["past"], case["past"] + n, device=DEVICE)
        pages = s["table"][i].long()[p // page]
        k_cache[pages, p % page] = turned[at:at + n, h:]
        v_cache[pages, p % page] = x[at:at + n, h + kv:]
        at += n
    return {"q": turned[:, :h].contiguous(), "k_cache": k_cache, "v_cache": v_cache}


def _exact_prompt(s, case):
    outs, lses, at = [], [], 0
    for i, n in enumerate(_lengths(case["seqs"], case["lo"], case["hi"])):
        count = n + case["past"]
        k, v = (_rows_of(x, s["table"][i], count, case["page"]).transpose(0, 1) for x in (s["k_cache"], s["v_cache"]))
        limit = case["past"] + 1 + torch.arange(n, device=DEVICE)
        out, lse = _softmax_of(s["q"][at:at + n].double().transpose(0, 1), k, v, limit)
        outs.append(out.transpose(0, 1))
        lses.append(lse.T)
        at += n
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def _exact_decode(s, case):
    prefixes = _lengths(case["groups"], case["prefix_lo"], case["prefix_hi"])
    group = [g for g, n in enumerate(_group_sizes(case)) for _ in range(n)]
    shared = [tuple(_rows_of(x, s["prefix_table"][g], p, case["page"]) for x in (s["k_cache"], s["v_cache"]))
              for g, p in enumerate(prefixes)]
    outs, lses = [], []
    for i, n in enumerate(_lengths(case["seqs"], case["lo"], case["hi"])):
        k, v = (_rows_of(x, s["table"][i], n, case["page"]) for x in (s["k_cache"], s["v_cache"]))
        if group:
            k, v = torch.cat([shared[group[i]][0], k]), torch.cat([shared[group[i]][1], v])
        kv = k.shape[1]
        q = s["q"][i].double().view(kv, -1, case["dim"])
        z = torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(case["dim"])
        lse = torch.logsumexp(z, dim=2)
        outs.append(torch.einsum("hgn,nhd->hgd", torch.exp(z - lse[..., None]), v).flatten(0, 1))
        lses.append(lse.flatten())
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}
