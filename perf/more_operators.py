"""The operators of a paged KV cache, as a serving program calls them. Kinds:

  rope    rope: rotary positions of q and k heads, half or interleaved pairs, the whole head or part of it, frequencies as
          they are or scaled for long contexts
  store   rope_store (or paged_store) + paged_load: a step's q normed and rotated, its k and v put into pages of bf16 or of
          8 bits, and the values the pages then stand for
  paged   gqa_paged: causal attention of the new tokens of every row, one or many and not as many in each, over its pages

A cache holds pages of page_size positions; row b's positions lie in the pages page_table[b], in their order, and its new
tokens are its last: q_start[b] .. q_start[b + 1] - 1 of the batch's tokens, at positions up to seq_lens[b] - 1. What lies
behind a row's length is memory that nothing has written yet (NaN here), and the table's entries there are -1. In a cache of 8
bits the vector of a (position, head) is D codes of four exponent and three mantissa bits (e4m3) and one byte E that stands
for the scale 2^(E - 127).
"""
import math
import random
import types

import torch

own = False

DEV = "cuda:0"
BF16 = torch.bfloat16
F8 = torch.float8_e4m3fn
EPS = 1e-6


def listed():
    return [
        # a guidance pair's decode step: the smallest call, latency only
        dict(name="rope_step", kind="rope", tokens=2, heads=40, head_dim=128, rotary=128, interleaved=False, scaling="none",
             reach=2048),
        # a long prompt far into a context that its frequencies were stretched for; half of each head, interleaved pairs
        dict(name="rope_prompt_far", kind="rope", tokens=4097, heads=40, head_dim=128, rotary=64, interleaved=True,
             scaling="yarn", reach=262144),
        # the new token of every row of a batch, into 8 bits
        dict(name="store_step_b16", kind="store", batch=16, heads=16, kv_heads=8, head_dim=128, page=16, bits=8, lo=1, hi=1,
             past=4000, norm=True, rope=True, interleaved=False),
        # chunks of a few prompts
        dict(name="store_prompts", kind="store", batch=4, heads=16, kv_heads=8, head_dim=128, page=64, bits=16, lo=700,
             hi=2047, past=1000, norm=True, rope=True, interleaved=False),
        # keys and values that are rotated already, or carry no positions, into 8 bits
        dict(name="store_plain_8bit", kind="store", batch=3, heads=0, kv_heads=4, head_dim=64, page=32, bits=8, lo=300,
             hi=1501, past=0, norm=False, rope=False, interleaved=False),
        # a guidance pair's decode step
        dict(name="paged_pair", kind="paged", batch=2, kv_heads=8, group=2, head_dim=128, page=16, bits=16, lo=1024, hi=1024,
             tlo=1, thi=1, few=0),
        # a server's ragged decode batch, 8 bits
        dict(name="paged_ragged_b32_8bit", kind="paged", batch=32, kv_heads=8, group=2, head_dim=128, page=32, bits=8, lo=300,
             hi=8192, tlo=1, thi=1, few=0),
        # long rows, a large group (32 q / 4 KV heads)
        dict(name="paged_long_g8", kind="paged", batch=4, kv_heads=4, group=8, head_dim=128, page=64, bits=16, lo=20001,
             hi=32768, tlo=1, thi=1, few=0),
        # one to five tokens a row to verify, head_dim 64
        dict(name="paged_verify", kind="paged", batch=8, kv_heads=8, group=4, head_dim=64, page=16, bits=16, lo=700, hi=8192,
             tlo=1, thi=5, few=0),
        # a server's mixed step: six rows decode, two are chunks of a prompt
        dict(name="paged_mixed", kind="paged", batch=8, kv_heads=8, group=2, head_dim=128, page=16, bits=16, lo=900, hi=5000,
             tlo=333, thi=500, few=6),
        # a chunk behind a long context, 8 bits
        dict(name="paged_chunk_8bit", kind="paged", batch=1, kv_heads=8, group=2, head_dim=128, page=128, bits=8, lo=16384,
             hi=16384, tlo=512, thi=512, few=0),
        # the prefill of a long prompt
        dict(name="paged_prefill_8k", kind="paged", batch=1, kv_heads=8, group=2, head_dim=128, page=64, bits=16, lo=8192,
             hi=8192, tlo=8192, thi=8192, few=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "store", "store", "paged", "paged", "paged", "paged"])
    D = rng.choice([64, 128])
    if kind == "rope":
        return dict(kind=kind, tokens=_log(rng, 1, 8192), heads=rng.randint(1, 40), head_dim=D,
                    rotary=rng.choice([D, D, D // 2, 16 * rng.randint(1, D // 16)]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), reach=_log(rng, 8192, 1048576))
    page, bits = rng.choice([16, 32, 64, 128, 256]), rng.choice([8, 16])
    NKV = rng.choice([1, 2, 4, 8])
    if kind == "store":
        hi = _log(rng, 1, 2047)
        rope = rng.random() < 0.75
        return dict(kind=kind, batch=rng.randint(1, 8), heads=NKV * rng.choice([1, 2, 4]) if rope else 0, kv_heads=NKV, head_dim=D,
                    page=page, bits=bits, lo=max(1, hi // 3), hi=hi, past=rng.choice([0, rng.randint(1, 5000)]),
                    norm=rope and rng.random() < 0.5, rope=rope, interleaved=rng.random() < 0.5)
    c = dict(kind=kind, kv_heads=NKV, group=rng.choice([1, 2, 4, 8]), head_dim=D, page=page, bits=bits, few=0)
    form = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
    if form == "decode":
        hi = _log(rng, 64, 32768)
        return c | dict(batch=_log(rng, 1, 32 if hi <= 8192 else 4), lo=max(1, hi // 4), hi=hi, tlo=1, thi=1)
    if form == "verify":
        hi = _log(rng, 64, 16384)
        return c | dict(batch=rng.randint(1, 8), lo=max(8, hi // 4), hi=hi, tlo=1, thi=rng.randint(2, 8))
    c |= dict(kv_heads=min(NKV, 4), group=min(c["group"], 4))
    T, past = _log(rng, 16, 1500), rng.choice([0, _log(rng, 1, 8192)])
    if form == "chunk":
        return c | dict(batch=rng.randint(1, 2), lo=T + past, hi=T + past, tlo=max(1, T // 2), thi=T)
    few = rng.randint(1, 6)
    return c | dict(batch=few + 1, lo=T + past // 2, hi=T + past, tlo=T, thi=T, few=few)


# ------------------------------------------------------------------------------------------------------- inputs

def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _rows(case, seed):
    """Each row's length and its number of new tokens (a batch is of one size whatever the seed)."""
    r, size = random.Random(seed * 7919 + 17), random.Random(case["batch"] * 7919 + case["hi"])
    B = case["batch"]
    if case["kind"] == "store":
        new = [size.randint(case["lo"], case["hi"]) for _ in range(B)]
        new[0] = case["hi"]
        return [n + r.randint(case["past"] // 2, case["past"]) for n in new], new
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(B)]
    lens[0] = case["hi"]
    new = [1 if b >= B - case["few"] else min(case["lo"], size.randint(case["tlo"], case["thi"])) for b in range(B)]
    new[0] = case["thi"]
    return lens, new


def _scale_exponent(x):
    """E - 127 of the smallest scale 2^(E - 127), E >= 10, with max |x| <= 448 scale; x [..., D] in 32 bits."""
    f, e = torch.frexp(x.abs().amax(-1))  # f in [0.5, 1); 448 = 0.875 2^9
    e = torch.where(f > 0.875, e - 8, e - 9)
    return torch.where(f == 0, torch.full_like(e, -117), e).clamp(min=-117)


def _pack(x):
    """(codes, scales) of x [..., D]: codes are x / scale rounded to the nearest e4m3 value, ties to the even code."""
    x = x.float()
    e = _scale_exponent(x)
    return (x * torch.exp2(-e.double()).float()[..., None]).to(F8), (e + 127).to(torch.uint8)


def _inverse_frequencies(R, scaling, base=1e6):
    """(frequencies [R / 2] in 64 bits, what cos and sin are multiplied by), for contexts 8 times 32768."""
    i = torch.arange(0, R, 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * 8.0 ** (R / max(R - 2, 1))
    f = base ** (-i / R)
    if scaling == "linear":
        f = f / 8
    if scaling != "yarn":
        return f, 1.0
    turns = [R * math.log(32768 / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32, 1)]
    low, high = max(math.floor(turns[0]), 0), min(math.ceil(turns[1]), R - 1)
    ramp = ((torch.arange(R // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    return f / 8 * ramp + f * (1 - ramp), 0.1 * math.log(8) + 1


def _pages(s, g, lens):
    """A page table whose pages are spread over the cache at random, -1 behind each row's last."""
    width = max(-(-n // s.page) for n in lens)
    count = [-(-n // s.page) for n in lens]
    s.pages = sum(count) + 3
    order = torch.randperm(s.pages, generator=g, device=DEV, dtype=torch.int32)
    table = torch.full((s.batch, width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(count):
        table[b, :n] = order[at:at + n]
        at += n
    s.table = table


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    s = types.SimpleNamespace(**{k: v for k, v in case.items() if k != "name"})
    D = s.head_dim
    if s.kind == "rope":
        # q and k heads of a projection's output, the values behind them
        s.x = _randn(g, s.tokens, s.heads + 2, D).to(BF16)[:, :s.heads]
        s.positions = torch.randint(0, s.reach, (s.tokens,), generator=g, device=DEV)
        f, s.factor = _inverse_frequencies(s.rotary, s.scaling)
        s.inv_freq = f.to(DEV)
        return s
    H = s.kv_heads
    lens, new = _rows(case, seed)
    s.lens, s.total, s.most, s.longest = _ints(lens), sum(new), max(new), max(lens)
    s.q_start = _ints([sum(new[:b]) for b in range(s.batch + 1)])
    s.first = s.lens - _ints(new)
    _pages(s, g, lens)
    P = s.page
    if s.kind == "store":
        qkv = _randn(g, s.total, s.heads + 2 * H, D).to(BF16)
        s.q, s.k, s.v = qkv.split([s.heads, H, H], 1)
        f, s.factor = _inverse_frequencies(D, "none")
        s.inv_freq = f.to(DEV)
        s.weights = [(1 + 0.2 * _randn(g, D)).to(BF16) for _ in range(2)] if s.norm else [None, None]
        s.cache = [torch.zeros(s.pages, H, P, D, dtype=torch.uint8, device=DEV).view(F8) if s.bits == 8 else
                   torch.zeros(s.pages, H, P, D, dtype=BF16, device=DEV) for _ in range(2)]
        s.cache += [torch.full((s.pages, H, P), 10, dtype=torch.uint8, device=DEV) if s.bits == 8 else None for _ in range(2)]
        return s
    hot = torch.rand(s.pages, H, P, 1, generator=g, device=DEV) < 0.01  # keys that stand out, as trained heads have them
    k, v = _randn(g, s.pages, H, P, D), _randn(g, s.pages, H, P, D)
    k = torch.where(hot, 4 * k, k)
    behind = torch.ones(s.pages, P, dtype=torch.bool, device=DEV)  # what no row holds
    pos = torch.arange(s.table.size(1) * P, device=DEV)
    inside = (pos < s.lens[:, None]).view(s.batch, -1, P)
    behind[s.table.long()[s.table >= 0]] = ~inside[s.table >= 0]
    behind = behind[:, None]
    if s.bits == 8:
        (kc, ks), (vc, vs) = _pack(k.to(BF16)), _pack(v.to(BF16))
        s.cache = [kc, vc, ks.masked_fill(behind, 255), vs.masked_fill(behind, 255)]
    else:
        s.cache = [x.to(BF16).masked_fill(behind[..., None], float("nan")) for x in (k, v)] + [None, None]
    s.q = (1.5 * _randn(g, s.total, H * s.group, D)).to(BF16)
    s.scale = D ** -0.5
    return s


# ------------------------------------------------------------------------------------------------- the plain forms

def _rotate(x, positions, inv_freq, factor, interleaved):
    """x [N, H, D] in 32 bits; the angles in 64, as far positions need."""
    R = 2 * inv_freq.numel()
    a = positions.double()[:, None] * inv_freq
    cos, sin = ((factor * t).float()[:, None] for t in (a.cos(), a.sin()))
    r, rest = x[..., :R], x[..., R:]
    if interleaved:
        x0, x1 = r[..., 0::2], r[..., 1::2]
        y = torch.stack((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1).flatten(-2)
    else:
        x0, x1 = r.chunk(2, -1)
        y = torch.cat((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1)
    return torch.cat((y, rest), -1)


def _norm(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _values(codes, scales):
    return codes.float() * torch.exp2(scales.float() - 127)[..., None]


def _token_rows(s):
    """(row, position) of each of the batch's tokens."""
    n = torch.arange(s.total, device=DEV)
    row = torch.searchsorted(s.q_start[1:], n.int(), right=True)
    return row, s.first[row] + n - s.q_start[row]


def _plain_store(s):
    row, pos = _token_rows(s)
    q, k, v = s.q.float(), s.k.float(), s.v.float()
    if s.rope:
        q, k = (_rotate(_norm(x, w), pos, s.inv_freq, s.factor, s.interleaved) for x, w in ((q, s.weights[0]), (k, s.weights[1])))
    page, at = s.table[row, pos // s.page].long(), (pos % s.page).long()
    for i, x in enumerate((k, v)):
        if s.bits == 8:
            codes, scales = _pack(x)
            s.cache[i].view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
            s.cache[2 + i][page, :, at] = scales
        else:
            s.cache[i][page, :, at] = x.to(BF16)
    # the new tokens of every row read back, as many as the longest has; zeros behind the row's last page
    p = s.first[:, None] + torch.arange(s.most, device=DEV)
    there = p < s.table.size(1) * s.page
    page = s.table.gather(1, (p // s.page).clamp(max=s.table.size(1) - 1).long())
    there &= page >= 0
    page, at = page.clamp(min=0).long(), (p % s.page).long()
    back = []
    for i in range(2):
        x = s.cache[i].view(torch.uint8)[page, :, at].view(F8) if s.bits == 8 else s.cache[i][page, :, at]
        x = _values(x, s.cache[2 + i][page, :, at]) if s.bits == 8 else x
        back.append(torch.where(there[..., None, None], x, 0).to(BF16).transpose(1, 2).contiguous())
    return (q.to(BF16), *back) if s.rope else tuple(back)


def _plain_paged(s):
    """Every row's pages side by side, its tokens padded to the longest chunk, a mask, and a softmax in 32 bits."""
    B, H, D, G, T, C = s.batch, s.kv_heads, s.head_dim, s.group, s.most, s.table.size(1) * s.page
    inside = (torch.arange(C, device=DEV) < s.lens[:, None])[:, None, :, None]
    kv = []
    for i in range(2):
        at = s.table.clamp(min=0).long()
        x = s.cache[i].view(torch.uint8)[at].view(F8) if s.bits == 8 else s.cache[i][at]
        x = _values(x, s.cache[2 + i][at]) if s.bits == 8 else x.float()
        kv.append(torch.where(inside, x.transpose(1, 2).reshape(B, H, C, D), 0))
    row, pos = _token_rows(s)
    t = pos - s.first[row]
    q = torch.zeros(B, T, H, G, D, device=DEV)
    q[row, t] = s.q.float().view(-1, H, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(B, H, G * T, D)
    last = s.first[:, None] + torch.arange(T, device=DEV)
    ok = torch.arange(C, device=DEV) <= last[..., None]
    x = (q @ kv[0].transpose(2, 3)).view(B, H, G, T, C)
    x = torch.where(ok[:, None, None], x * s.scale, float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    out = (x.view(B, H, G * T, C) @ kv[1]).view(B, H, G, T, D)
    return out.permute(0, 3, 1, 2, 4).reshape(B, T, H * G, D)[row, t].to(BF16)


def run(s):
    if own:
        return _own(s)
    if s.kind == "rope":
        return _rotate(s.x.float(), s.positions, s.inv_freq, s.factor, s.interleaved).to(BF16)
    return _plain_store(s) if s.kind == "store" else _plain_paged(s)


# ------------------------------------------------------------------------------------------- the framework's calls

def _package():
    import __graft_entry__

    return __graft_entry__.package()


def _own(s):
    pkg = _package()
    if s.kind == "rope":
        return pkg.rope(s.x, s.positions, pkg.Rope(s.inv_freq, s.factor, s.interleaved))
    cache = pkg.PagedCache(*s.cache)
    if s.kind == "store":
        if s.rope:
            q = pkg.rope_store(s.q, s.k, s.v, cache, s.table, s.lens, pkg.Rope(s.inv_freq, s.factor, s.interleaved), s.q_start,
                               q_norm_weight=s.weights[0], k_norm_weight=s.weights[1], eps=EPS)
            return (q, *pkg.paged_load(cache, s.table, s.first, s.most))
        pkg.paged_store(s.k, s.v, cache, s.table, s.lens, s.q_start)
        return pkg.paged_load(cache, s.table, s.first, s.most)
    q_start = None if s.most == 1 else s.q_start
    return pkg.gqa_paged(s.q, cache, s.table, s.lens, s.scale, q_start, max_tokens=s.most, max_seq_len=s.longest)


# -------------------------------------------------------------------------------------------------- what it costs

def work(case):
    """Queries, outputs and the rows' keys and values once; 2 D flops per product of a (query, position) pair. Lengths and
    numbers of tokens are taken at the middle of their ranges."""
    D = case["head_dim"]
    if case["kind"] == "rope":
        return {"bytes": case["tokens"] * (4 * case["heads"] * D + 8), "flops": 0}
    B, H = case["batch"], case["kv_heads"]
    row = D + 1 if case["bits"] == 8 else 2 * D
    if case["kind"] == "store":
        n = case["hi"] + (B - 1) * (case["lo"] + case["hi"]) / 2
        back = case["hi"] * B  # read back and written as bf16
        return {"bytes": n * (4 * case["heads"] * D + 4 * H * D + 2 * H * row) + back * 2 * H * (row + 2 * D), "flops": 0}
    G, few = case["group"], case["few"]
    n = case["hi"] + (B - 1) * (case["lo"] + case["hi"]) / 2
    rest = (case["lo"] + case["hi"]) / 2
    chunks = B - few
    T = case["thi"] + (chunks - 1) * (case["tlo"] + case["thi"]) / 2  # tokens of the rows that have many
    t = T / chunks
    pairs = T * ((n - few * rest) / chunks - (t - 1) / 2) + few * rest
    return {"bytes": 2 * n * H * row + 4 * (T + few) * H * G * D, "flops": 4 * D * pairs * H * G}


# ----------------------------------------------------------------------------------- the definitions in 64 bits

def _exact_turn(x, positions, inv_freq, factor, interleaved):
    """Each pair as a complex number, multiplied by factor e^(i angle)."""
    n = inv_freq.numel()
    at = torch.arange(n, device=DEV)
    first, second = (2 * at, 2 * at + 1) if interleaved else (at, at + n)
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.full_like(inv_freq, factor), torch.outer(positions.double(), inv_freq))[:, None]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_round(x):
    """Each vector at the smallest power of two that keeps its largest magnitude within 448, every value at the nearest of
    those of three mantissa bits and exponents from 2^-6 on; of two as near, the even one."""
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.full_like(top, 2.0 ** -117)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):
        scale = torch.where(top > 448 * scale * 2.0 ** (step - 1), scale * 2.0 ** step, scale)
    a = x / scale
    unit = torch.exp2(torch.frexp(a.abs().clamp(min=2.0 ** -6)).exponent.float() - 4).double()
    return torch.round(a / unit) * unit * scale  # (round: ties to even)


def _exact_store(s):
    row, pos = _token_rows(s)
    q, k, v = s.q.double(), s.k.double(), s.v.double()
    if s.rope:
        turned = []
        for x, w in ((q, s.weights[0]), (k, s.weights[1])):
            if w is not None:
                x = w.double() * x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.size(-1) + EPS)
            turned.append(_exact_turn(x, pos, s.inv_freq, s.factor, s.interleaved))
        q, k = turned
    back = []
    for x in (k, v):
        if s.bits == 8:
            x = _exact_round(x)
        y = torch.zeros(s.batch, s.kv_heads, s.most, s.head_dim, dtype=torch.float64, device=DEV)
        y[row, :, (pos - s.first[row]).long()] = x
        back.append(y)
    return (q, *back) if s.rope else tuple(back)


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "rope":
        return _exact_turn(s.x.double(), s.positions, s.inv_freq, s.factor, s.interleaved)
    if s.kind == "store":
        return _exact_store(s)
    H, G, D, P = s.kv_heads, s.group, s.head_dim, s.page
    out = torch.zeros(s.total, H * G, D, dtype=torch.float64, device=DEV)
    starts = s.q_start.tolist()
    for b, n in enumerate(s.lens.tolist()):
        pages = s.table[b, :-(-n // P)].long()
        t0, t1 = starts[b], starts[b + 1]
        future = torch.arange(n, device=DEV)[None] > torch.arange(n - (t1 - t0), n, device=DEV)[:, None]
        for h in range(H):
            k, v = (x[pages, h].double().reshape(-1, D)[:n] for x in s.cache[:2])
            if s.bits == 8:
                k, v = (x * 2.0 ** (e[pages, h].reshape(-1)[:n].double() - 127)[:, None] for x, e in zip((k, v), s.cache[2:]))
            for i in range(h * G, h * G + G):
                e = (s.q[t0:t1, i].double() @ k.t() / math.sqrt(D)).masked_fill_(future, -math.inf)
                out[t0:t1, i] = torch.softmax(e, -1) @ v
    return out
