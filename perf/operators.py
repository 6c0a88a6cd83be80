"""The operators that keep a long KV cache small and read it, as a serving program calls them. Kinds:

  window  gqa_window: causal attention of T query tokens over a sliding window and the row's first positions (sinks),
          from one token (a decode step) to a long chunk (prefill), on a bf16 cache
  store   kv4_store + kv4_load: new k / v rounded into a 4-bit cache, and the values it then stands for
  kv4     gqa_decode_kv4: decode attention over a 4-bit cache
  track   gqa_decode_tracked: a decode step that also adds its attention weights to the cache's weights
  evict   kv_evict: the positions with the largest accumulated weights kept, and the cache compacted to them

A row b of a cache holds positions [start[b], lens[b]); the T query tokens of a row are its last T positions. What lies
behind a row's length is memory that nothing has written yet (NaN here). A 4-bit cache holds, for each 32 consecutive
dims, 32 codes of one sign, two exponent and one mantissa bit (two to a byte, the even dim in the low half) and one byte
E that stands for the scale 2^(E - 127).
"""
import math
import random
import types

import torch

own = False

DEV = "cuda:0"
BF16 = torch.bfloat16
F4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # a CFG pair's decode step past its window: the smallest call, latency only
        dict(name="window_step", kind="window", batch=2, kv_heads=8, group=2, head_dim=128, capacity=4096, tokens=1,
             lo=2900, hi=2900, window=1024, sinks=4),
        # a server's ragged batch over long rows, some still shorter than the window
        dict(name="window_ragged_b16", kind="window", batch=16, kv_heads=8, group=2, head_dim=128, capacity=16384,
             tokens=1, lo=500, hi=16384, window=4096, sinks=4),
        # a chunk of a chunked prefill behind earlier context, left-padded rows, odd sizes, head_dim 64
        dict(name="window_chunk_333", kind="window", batch=3, kv_heads=4, group=4, head_dim=64, capacity=2600,
             tokens=333, lo=1500, hi=2501, window=777, sinks=5),
        # the prefill of a long prompt
        dict(name="window_prefill_8k", kind="window", batch=1, kv_heads=8, group=2, head_dim=128, capacity=8192,
             tokens=8192, lo=8192, hi=8192, window=4096, sinks=16),
        # the new token of every row of a batch
        dict(name="store_step_b16", kind="store", batch=16, kv_heads=8, head_dim=128, capacity=4096, tokens=1),
        # a prompt's keys and values
        dict(name="store_prompt", kind="store", batch=4, kv_heads=8, head_dim=128, capacity=4096, tokens=2047),
        # a CFG pair at serving shape
        dict(name="kv4_pair_1k", kind="kv4", batch=2, kv_heads=8, group=2, head_dim=128, capacity=2048, tokens=1,
             lo=1024, hi=1024, window=0, sinks=0),
        # a few tokens a row to verify over a ragged batch with a window
        dict(name="kv4_verify_window", kind="kv4", batch=8, kv_heads=8, group=4, head_dim=64, capacity=8192, tokens=3,
             lo=700, hi=8192, window=4096, sinks=4),
        # a larger group over a long context (32 q / 4 KV heads)
        dict(name="kv4_long_32k_g8", kind="kv4", batch=4, kv_heads=4, group=8, head_dim=128, capacity=32768, tokens=1,
             lo=20001, hi=32768, window=0, sinks=0),
        # a CFG pair's decode step with its weights accumulated
        dict(name="track_pair", kind="track", batch=2, kv_heads=8, group=2, head_dim=128, capacity=2048, lo=1377,
             hi=1377),
        # the same over a batch of long rows
        dict(name="track_long_b4_g4", kind="track", batch=4, kv_heads=8, group=4, head_dim=128, capacity=16384,
             lo=9000, hi=16384),
        # a batch that reached its budget: half of each row goes
        dict(name="evict_b4_8k", kind="evict", batch=4, kv_heads=8, head_dim=128, capacity=8192, lo=7000, hi=8192,
             keep=4096, sinks=4, recent=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "store", "kv4", "kv4", "track", "evict"])
    D = rng.choice([64, 128])
    NKV = rng.choice([1, 2, 4, 8])
    if kind == "store":
        return dict(kind=kind, batch=rng.randint(1, 8), kv_heads=NKV, head_dim=D, capacity=4096,
                    tokens=_log(rng, 1, 2047))
    if kind == "evict":
        cap = _log(rng, 200, 16384)
        keep = rng.randint(64, cap - 60)
        return dict(kind=kind, batch=rng.randint(1, 4), kv_heads=NKV, head_dim=D, capacity=cap, lo=cap // 2, hi=cap,
                    keep=keep, sinks=rng.randint(0, 8), recent=rng.randint(0, keep // 2))
    G = rng.choice([1, 2, 4, 8])
    if kind == "track":
        cap = _log(rng, 64, 16384)
        return dict(kind=kind, batch=rng.randint(1, 4), kv_heads=NKV, group=G, head_dim=D, capacity=cap,
                    lo=max(1, cap // 3), hi=cap)
    c = dict(kind=kind, kv_heads=NKV, group=G, head_dim=D, window=0, sinks=0)
    if kind == "kv4":
        cap = _log(rng, 64, 32768)
        c |= dict(batch=rng.randint(1, 4), capacity=cap, tokens=rng.choice([1, 1, 1, 2, 3, 5]), lo=max(8, cap // 4), hi=cap)
        if rng.random() < 0.5:
            c |= dict(window=_log(rng, 16, 4096), sinks=rng.randint(0, 8))
        return c
    if rng.random() < 0.5:  # a decode step, or a few tokens
        cap = _log(rng, 64, 16384)
        c |= dict(batch=_log(rng, 1, 16), capacity=cap, tokens=rng.choice([1, 1, 1, 2, 4]), lo=max(8, cap // 4), hi=cap)
    else:  # a chunk
        T = _log(rng, 16, 2048)
        past = rng.choice([0, rng.randint(1, 4096)])
        c |= dict(batch=rng.randint(1, 2), kv_heads=min(NKV, 4), group=min(G, 4), capacity=T + past + rng.randint(0, 99),
                  tokens=T, lo=T + past, hi=T + past)
    return c | dict(window=_log(rng, 16, 4096), sinks=rng.randint(0, 16))


# ------------------------------------------------------------------------------------------------------- inputs

def _lengths(case, seed):
    """Row lengths spread over [lo, hi], and the left padding of every third row."""
    r = random.Random(seed * 7919 + 17)
    B, lo, hi = case["batch"], case["lo"], case["hi"]
    lens = [r.randint(lo, hi) for _ in range(B)]
    lens[0] = hi
    start = [r.randint(0, max(0, (n - case.get("tokens", 1)) // 8)) if b % 3 == 2 else 0 for b, n in enumerate(lens)]
    return lens, start


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _keys(g, *shape):
    """Keys with a few positions that stand out, as trained heads have them."""
    hot = torch.rand(shape[0], shape[1], shape[2], 1, generator=g, device=DEV) < 0.01
    k = _randn(g, *shape)
    return torch.where(hot, 4 * k, k).to(BF16)


def _pack(x):
    """(codes, scales) of x [..., D] bf16: the scale's exponent is floor(log2(amax)) - 2, one more where amax is over
    1.75 times a power of two; codes are x / scale rounded to the nearest value of F4, ties to the even code."""
    b = x.float().unflatten(-1, (-1, 32))
    f, e = torch.frexp(b.abs().amax(-1))  # f in [0.5, 1)
    e = torch.where(f > 0.875, e - 2, e - 3).clamp(-126, 127)
    e = torch.where(f == 0, torch.full_like(e, -126), e)
    y = b / torch.exp2(e.double()).float()[..., None]
    a = y.abs()
    # codes 0 .. 7 stand for 0 .5 1 1.5 2 3 4 6; a border goes to the even code
    c = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int()
         + (a > 5).int())
    c = (c | (y < 0).int() * 8).flatten(-2)
    return (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8), (e + 127).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    s = types.SimpleNamespace(**{k: v for k, v in case.items() if k != "name"})
    B, H, D, C = s.batch, s.kv_heads, s.head_dim, s.capacity
    s.scale = D ** -0.5
    if s.kind == "store":
        s.k, s.v = _keys(g, B, H, s.tokens, D), _randn(g, B, H, s.tokens, D).to(BF16)
        r = random.Random(seed)
        s.slots = _ints([r.randint(0, C - s.tokens) for _ in range(B)])
        s.cache = [torch.zeros(B, H, C, w, dtype=torch.uint8, device=DEV) for w in (D // 2, D // 2, D // 32, D // 32)]
        return s
    lens, start = _lengths(case, seed)
    s.lens, s.start = _ints(lens), _ints(start)
    s.longest = case["hi"]
    behind = (torch.arange(C, device=DEV) >= s.lens[:, None])[:, None, :, None]
    k, v = _keys(g, B, H, C, D), _randn(g, B, H, C, D).to(BF16)
    if s.kind == "kv4":
        (kc, ks), (vc, vs) = _pack(k), _pack(v)
        s.cache = [kc, vc, ks.masked_fill(behind, 255), vs.masked_fill(behind, 255)]
    else:
        s.k, s.v = k.masked_fill(behind, float("nan")), v.masked_fill(behind, float("nan"))
    if s.kind in ("track", "evict"):  # sums of probabilities; small ones often equal
        w = torch.exp(2 * _randn(g, B, H, C) - 3)
        s.weights = torch.where(w < 0.05, torch.floor(w * 256) / 256, w).masked_fill(behind[..., 0], 0)
        s.weights_out = torch.zeros_like(s.weights)
    if s.kind == "evict":
        s.outs = [torch.zeros_like(s.k), torch.zeros_like(s.v)]
        return s
    T = case.get("tokens", 1)
    s.q = (1.5 * _randn(g, B, H * s.group, T, D)).to(BF16)
    if s.kind == "track":
        s.q = s.q[:, :, 0].contiguous()
    return s


# ------------------------------------------------------------------------------------------------- the plain forms

def _visible(lens, start, T, C, window, sinks):
    """[B, T, C]: which positions each query token attends."""
    p = torch.arange(C, device=DEV)
    end = (lens[:, None] - (T - 1) + torch.arange(T, device=DEV))[:, :, None]
    ok = (p < end) & (p >= start[:, None, None])
    if window > 0:
        ok &= (p >= end - window) | (p < (start + sinks)[:, None, None])
    return ok


def _attend(q, k, v, ok, scale):
    """(out [B, NH, T, D], probabilities [B, NKV, G, T, C]) of q [B, NH, T, D] over k, v [B, NKV, C, D]; out is 0 where
    a token attends nothing."""
    B, NH, T, D = q.shape
    H, C = k.size(1), k.size(2)
    used = ok.any(1)[:, None, :, None]
    k, v = torch.where(used, k, 0), torch.where(used, v, 0)
    x = (q.reshape(B, H, NH // H * T, D) @ k.transpose(2, 3)).view(B, H, NH // H, T, C)
    x = torch.where(ok[:, None, None], x * scale, float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    x = x / x.sum(-1, keepdim=True).clamp(min=1e-30)
    return (x.view(B, H, -1, C) @ v).view(B, NH, T, D), x


def _unpack(codes, scales):
    """The values of a 4-bit cache, in 32 bits."""
    table = torch.tensor(F4 + [-x for x in F4], device=DEV)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    x = table[c.int()].unflatten(-1, (-1, 32))
    e = scales.float()[..., None]
    return torch.where(e == 255, float("nan"), x * torch.exp2(e - 127)).flatten(-2)


def _slots(s):
    t = (s.slots[:, None].long() + torch.arange(s.tokens, device=DEV))[:, None, :, None]
    return t.expand(-1, s.kv_heads, -1, -1)


def _plain_store(s):
    at = _slots(s)
    (kc, ks), (vc, vs) = _pack(s.k), _pack(s.v)
    for to, x in zip(s.cache, (kc, vc, ks, vs)):
        to.scatter_(2, at.expand(x.shape), x)
    kc, vc, ks, vs = (c.gather(2, at.expand(-1, -1, -1, c.size(3))) for c in s.cache)
    return _unpack(kc, ks).to(BF16), _unpack(vc, vs).to(BF16)


def _plain_track(s):
    ok = _visible(s.lens, s.start, 1, s.capacity, 0, 0)
    out, p = _attend(s.q[:, :, None].float(), s.k.float(), s.v.float(), ok, s.scale)
    s.weights_out.copy_(torch.where(ok, s.weights + p[:, :, :, 0].sum(2), s.weights_out))
    return out[:, :, 0].to(BF16), s.weights_out


def _kept(s, weights):
    """(index [B, NKV, keep], lens [B]): the positions that stay, ascending, -1 behind the last."""
    C, keep = s.capacity, s.keep
    p = torch.arange(C, device=DEV)
    n = s.lens - s.start
    inside = (p >= s.start[:, None]) & (p < s.lens[:, None])
    always = inside & ((p < (s.start + s.sinks)[:, None]) | (p >= (s.lens - s.recent)[:, None]))
    w = torch.where(always[:, None], float("inf"), torch.where(inside[:, None], weights, float("-inf")))
    index = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    lens = n.clamp(max=keep)
    index = torch.where((torch.arange(index.size(-1), device=DEV) < lens[:, None])[:, None], index, C)
    index = torch.sort(index, dim=-1).values
    return torch.where(index == C, -1, index).int(), lens.int()


def _plain_evict(s):
    index, lens = _kept(s, s.weights)
    n = index.size(-1)
    at, there = index.long().clamp(min=0), index >= 0
    for to, x in zip(s.outs, (s.k, s.v)):
        rows = x.gather(2, at[..., None].expand(-1, -1, -1, x.size(3)))
        to[:, :, :n] = torch.where(there[..., None], rows, to[:, :, :n])
    # the weights move along; what a row gives up reads 0
    w = torch.zeros_like(s.weights)
    w[:, :, :n] = torch.where(there, s.weights.gather(2, at), 0)
    behind = torch.arange(s.capacity, device=DEV) >= s.lens[:, None]
    s.weights_out.copy_(torch.where(behind[:, None], s.weights_out, w))
    return (*s.outs, s.weights_out, index, lens)


def run(s):
    if own:
        return _own(s)
    if s.kind == "store":
        return _plain_store(s)
    if s.kind == "track":
        return _plain_track(s)
    if s.kind == "evict":
        return _plain_evict(s)
    ok = _visible(s.lens, s.start, s.tokens, s.capacity, s.window, s.sinks)
    if s.kind == "kv4":
        k, v = _unpack(s.cache[0], s.cache[2]), _unpack(s.cache[1], s.cache[3])
    else:
        k, v = s.k.float(), s.v.float()
    return _attend(s.q.float(), k, v, ok, s.scale)[0].to(BF16).transpose(1, 2).contiguous()


# ------------------------------------------------------------------------------------------- the framework's calls

def _package():
    import __graft_entry__

    return __graft_entry__.package()


def _own(s):
    pkg = _package()
    if s.kind == "window":
        return pkg.gqa_window(s.q, s.k, s.v, s.lens, s.scale, s.window, sinks=s.sinks, kv_start=s.start,
                              max_seq_len=s.longest).view(s.batch, s.tokens, -1, s.head_dim)
    if s.kind == "store":
        cache = pkg.Kv4Cache(*s.cache)
        pkg.kv4_store(s.k, s.v, cache, s.slots)
        return pkg.kv4_load(cache, s.slots, s.tokens)
    if s.kind == "kv4":
        return pkg.gqa_decode_kv4(s.q, pkg.Kv4Cache(*s.cache), s.lens, s.scale, kv_start=s.start, window=s.window,
                                  sinks=s.sinks, max_seq_len=s.longest).view(s.batch, s.tokens, -1, s.head_dim)
    if s.kind == "track":
        out = pkg.gqa_decode_tracked(s.q, s.k, s.v, s.lens, s.scale, s.weights, weights_out=s.weights_out,
                                     kv_start=s.start, max_seq_len=s.longest)
        return out, s.weights_out
    index, lens = pkg.kv_evict((s.k, s.v), s.weights, s.lens, s.keep, sinks=s.sinks, recent=s.recent,
                               kv_start=s.start, outs=s.outs, weights_out=s.weights_out)
    return (*s.outs, s.weights_out, index, lens)


# -------------------------------------------------------------------------------------------------- what it costs

def work(case):
    """The attended K and V rows, queries, outputs and weights once; 2 D flops per product of a (query, position)
    pair. Lengths are taken at the middle of their range."""
    B, H, D = case["batch"], case["kv_heads"], case["head_dim"]
    row = D // 2 + D // 32  # of one position and head in a 4-bit cache
    if case["kind"] == "store":  # bf16 in, codes out, and back
        return {"bytes": 2 * B * H * case["tokens"] * (4 * D + 2 * row), "flops": 0}
    n = (case["hi"] + (B - 1) * (case["lo"] + case["hi"]) / 2) / B
    if case["kind"] == "evict":
        kept = min(n, case["keep"])
        return {"bytes": B * H * (8 * n + kept * (2 * 2 * 2 * D + 4)), "flops": 0}
    T, NH = case.get("tokens", 1), H * case["group"]
    reach = case.get("window", 0) or n
    # positions that any token of the row attends, and (token, position) pairs
    seen = min(n, reach + T - 1 + case.get("sinks", 0))
    first, full = n - T + 1, min(n, reach + case.get("sinks", 0))
    short = max(0.0, min(T, full - first))  # tokens that still see less than the full reach
    pairs = short * (first + full) / 2 + (T - short) * full
    kv = 2 * row if case["kind"] == "kv4" else 4 * D
    more = 8 * n * H if case["kind"] == "track" else 0
    return {"bytes": B * (seen * H * kv + 4 * T * NH * D + more), "flops": B * pairs * NH * 4 * D}


# ----------------------------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    B, H, D, C = s.batch, s.kv_heads, s.head_dim, s.capacity
    if s.kind == "store":
        return tuple(_exact_round(x) for x in (s.k, s.v))
    if s.kind == "evict":
        return _exact_evict(s)
    lens, start = s.lens.tolist(), s.start.tolist()
    T, G = case.get("tokens", 1), s.group
    out = torch.zeros(B, T, H * G, D, dtype=torch.float64, device=DEV)
    weights = torch.zeros(B, H, C, dtype=torch.float64, device=DEV)
    for b in range(B):
        n0, n = start[b], lens[b]
        if n <= n0:
            continue
        pos = torch.arange(n0, n, device=DEV)[None]
        last = torch.arange(n - T, n, device=DEV)[:, None]  # each token's own position
        far = pos > last
        if case.get("window", 0):
            far |= (last - pos >= case["window"]) & (pos - n0 >= case["sinks"])
        for h in range(H):
            if s.kind == "kv4":
                k, v = (_exact_values(s.cache[i][b, h, n0:n], s.cache[i + 2][b, h, n0:n]) for i in (0, 1))
            else:
                k, v = s.k[b, h, n0:n].double(), s.v[b, h, n0:n].double()
            for g in range(G):
                q = s.q[b, h * G + g].double().view(T, D)
                e = (q @ k.t() / math.sqrt(D)).masked_fill_(far, -math.inf)
                e = torch.softmax(e, -1).nan_to_num_(0.0)
                out[b, :, h * G + g] = e @ v
                if s.kind == "track":
                    weights[b, h, n0:n] += e[0]
        if s.kind == "track":
            weights[b, :, n0:n] += s.weights[b, :, n0:n].double()
    return (out[:, 0], weights) if s.kind == "track" else out


def _exact_values(codes, scales):
    """Sign, exponent and mantissa of each code by arithmetic."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    sign, e, m = 1 - 2 * (c >> 3), (c >> 1) & 3, (c & 1).double()
    x = torch.where(e > 0, (1 + m / 2) * 2.0 ** (e - 1).clamp(min=0).double(), m / 2) * sign
    return x * torch.repeat_interleave(2.0 ** (scales.double() - 127), 32, -1)


def _exact_round(x):
    """Each block of 32 at the smallest power of two that keeps its largest magnitude within 7, every value at the
    nearest of the representable ones; of two as near, the one with the even code."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    scale = 2.0 ** torch.ceil(torch.log2(top / 7).clamp(min=-126))
    scale = torch.where(top > 7 * scale, 2 * scale, torch.where((top <= 3.5 * scale) & (scale > 2.0 ** -126), scale / 2, scale))
    a = (b / scale).abs()
    best, dist = torch.zeros_like(a), a.clone()
    for code, value in enumerate(F4[1:], 1):
        d = (a - value).abs()
        take = (d < dist) | ((d == dist) & (code % 2 == 0))
        best, dist = torch.where(take, value, best), torch.where(take, d, dist)
    return (best * torch.sign(b) * scale).flatten(-2)


def _exact_evict(s):
    """Row by row: the heaviest of the middle by (weight, position), the ends always."""
    B, H, C, keep = s.batch, s.kv_heads, s.capacity, s.keep
    outs = [torch.zeros_like(x, dtype=torch.float64) for x in (s.k, s.v)]
    weights = torch.zeros(B, H, C, dtype=torch.float64, device=DEV)
    index = torch.full((B, H, min(keep, C)), -1, dtype=torch.int32, device=DEV)
    lens = []
    for b, (n0, n) in enumerate(zip(s.start.tolist(), s.lens.tolist())):
        lens.append(min(n - n0, keep))
        for h in range(H):
            w = s.weights[b, h].tolist()
            at = list(range(n0, n))
            if n - n0 > keep:
                middle = at[s.sinks:len(at) - s.recent]
                middle = sorted(middle, key=lambda p: (-w[p], p))[:keep - s.sinks - s.recent]
                at = sorted(at[:s.sinks] + middle + at[len(at) - s.recent:])
            i = torch.tensor(at, device=DEV)
            index[b, h, :len(at)] = i
            weights[b, h, :len(at)] = s.weights[b, h, i].double()
            for to, x in zip(outs, (s.k, s.v)):
                to[b, h, :len(at)] = x[b, h, i].double()
    return (*outs, weights, index, torch.tensor(lens, dtype=torch.int32, device=DEV))
