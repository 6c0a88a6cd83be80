"""GPU: calls of the long-cache operators (include/bz_long_cache.h) that their documentation allows, or that they refuse, beyond
those of test_gpu_long_cache.py."""
import numpy as np
import pytest
import torch

import breeze_tts_2_flash_amd as pkg
from oracle.long_cache import attention_bound, window_attention

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def ints(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def randn(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(BF16)


# ------------------------------------------------------------------------------------------------- attention

@pytest.mark.parametrize("T,NKV,G", [(1, 2, 2), (5, 1, 4), (70, 8, 8), (300, 8, 2)])
@pytest.mark.parametrize("splits", [0, 3])
def test_scale_that_is_nan(device, T, NKV, G, splits):
    """It makes NaN of every token that attends a position; one that attends none still gets zeros."""
    rng = np.random.default_rng(T)
    D, cap = 128, T + 400
    q, k, v = (randn(rng, *s).to(device) for s in ((3, NKV * G, T, D), (3, NKV, cap, D), (3, NKV, cap, D)))
    lens, nan = ints([cap, T // 2, 0], device), float("nan")
    outs = [pkg.gqa_window(q, k, v, lens, nan, 100, sinks=3, num_splits=splits)]
    if T <= 16:
        cache = pkg.kv4_store(k, v, pkg.kv4_cache(3, NKV, cap, D, device), ints([0] * 3, device))
        outs.append(pkg.gqa_decode_kv4(q, cache, lens, nan, window=100, sinks=3, num_splits=splits))
    if T == 1:
        w = torch.zeros(3, NKV, cap, device=device)
        outs.append(pkg.gqa_decode_tracked(q, k, v, lens, nan, w, num_splits=splits))
        assert torch.isnan(w[0]).all() and (w[1:] == 0).all()
    for out in outs:
        out = out.view(3, T, -1)
        assert torch.isnan(out[0]).all() and (out[2] == 0).all()
        assert (out[1, :T - T // 2] == 0).all() and torch.isnan(out[1, T - T // 2:]).all()


@pytest.mark.parametrize("T,NKV,G,D", [(1, 2, 2, 128), (6, 1, 4, 64), (70, 8, 8, 64), (300, 8, 2, 128)])
@pytest.mark.parametrize("splits", [0, 4])
def test_scores_of_minus_infinity(device, T, NKV, G, D, splits):
    """Zeros where all a token attends scores -inf, and nothing of such a position where others score more."""
    rng = np.random.default_rng(T)
    n, window = T + 300, 90
    q, k, v = randn(rng, 1, NKV * G, T, D), randn(rng, 1, NKV, n, D), randn(rng, 1, NKV, n, D)
    q[..., 0], k[..., 0] = 1, 0
    clean = k.clone()
    half = n - T // 2 - 1  # the first tokens attend only positions before it
    k[:, :, :half, 0] = float("-inf")
    args = (ints([n], device), D ** -0.5, window)
    out = pkg.gqa_window(q.to(device), k.to(device), v.to(device), *args, num_splits=splits).view(T, NKV * G, D)
    end = n - T + 1 + torch.arange(T)
    none = end <= half
    assert none.any() or T == 1
    assert (out[none.to(device)] == 0).all() and (out[~none.to(device)] != 0).any(-1).all()
    # the others: as if the row began at `half`
    ref, spread, reach = window_attention(q.float(), clean.float(), v.float(), [n], D ** -0.5, window, 0, [half])
    late = (~none).numpy()
    excess = np.abs(out.float().cpu().numpy() - ref[0]) - attention_bound(ref, spread, reach, D ** -0.5, D, T > 16)[0]
    assert excess[late].max() <= 0
    if T == 1:
        k[..., 0] = float("-inf")
        kd, w = k.to(device), torch.rand(1, NKV, n, device=device)
        held = w.clone()
        for out in (pkg.gqa_window(q.to(device), kd, v.to(device), *args), pkg.gqa_decode(q[:, :, 0].to(device), kd, v.to(device), *args[:2]),
                    pkg.gqa_decode_tracked(q[:, :, 0].to(device), kd, v.to(device), *args[:2], w, num_splits=splits)):
            assert (out == 0).all()
        assert torch.equal(w, held)


@pytest.mark.parametrize("T,NKV,G,D,n,start,window,sinks", [
    (333, 4, 4, 64, 1501, 7, 777, 5), (200, 8, 4, 128, 300, 0, 90, 5), (200, 8, 4, 64, 300, 3, 60, 37), (250, 8, 2, 128, 900, 0, 500, 0),
    (130, 32, 8, 128, 500, 2, 100, 66), (200, 16, 8, 64, 700, 0, 33, 130), (800, 64, 2, 128, 1300, 1, 200, 4),
    (800, 64, 2, 64, 1100, 0, 222, 64),
])
@pytest.mark.parametrize("splits", [0, 3])
@pytest.mark.parametrize("value", [float("nan"), float("-inf")])
def test_positions_given_up_cost_a_chunk_nothing(device, T, NKV, G, D, n, start, window, sinks, splits, value):
    """What lies where no token looks (between the sinks and the window too) changes no bit of a chunk's output: it enters no
    product, and no column is worked out anew because of it."""
    from oracle.long_cache import attended
    rng = np.random.default_rng(T + n)
    q, k, v = (randn(rng, *s).to(device) for s in ((1, NKV * G, T, D), (1, NKV, n + 30, D), (1, NKV, n + 30, D)))
    args = dict(sinks=sinks, kv_start=ints([start], device), num_splits=splits)
    want = pkg.gqa_window(q, k, v, ints([n], device), D ** -0.5, window, **args)
    seen = set().union(*map(set, attended(start, n, T, window, sinks)))
    out = [p for p in range(n + 30) if p not in seen]
    assert any(start + sinks <= p < n for p in out)
    k[:, :, out], v[:, :, out] = value, value
    assert torch.equal(pkg.gqa_window(q, k, v, ints([n], device), D ** -0.5, window, **args), want)


# --------------------------------------------------------------------------------------------------- 4 bits

def test_kv4_refuses_overlaps(device):
    """Outputs, and the tensors of a cache that is written, which share memory with one another."""
    rng = np.random.default_rng(5)
    x, slot = randn(rng, 1, 2, 3, 128).to(device), ints([0], device)
    cache = pkg.kv4_cache(1, 2, 64, 128, device)
    rows = torch.zeros(1, 2, 80, 128, dtype=BF16, device=device)
    with pytest.raises(RuntimeError):
        pkg.kv4_load(cache, slot, 30, rows[:, :, :30], rows[:, :, 10:40])
    codes, scales = (torch.zeros(1, 2, 80, n, dtype=torch.uint8, device=device) for n in (64, 4))
    for bad in (cache._replace(k=codes[:, :, :64], v=codes[:, :, 16:]), cache._replace(k_scale=scales[:, :, :64], v_scale=scales[:, :, 16:]),
                cache._replace(k_scale=cache.k.view(1, 2, 1024, 4)[:, :, :64], v_scale=cache.v.view(1, 2, 1024, 4)[:, :, :64])):
        with pytest.raises(RuntimeError):
            pkg.kv4_store(x, x, bad, slot)


@pytest.mark.parametrize("D", [64, 128])
def test_kv4_cache_in_one_tensor(device, D):
    """A head's codes of K and V and their scales one behind the other in one tensor; outputs side by side."""
    rng = np.random.default_rng(D)
    B, NKV, cap, T = 2, 3, 40, 7
    at, room = [0, cap * D // 2, cap * D, cap * D + cap * D // 32], cap * (D + D // 16)
    one = torch.zeros(B, NKV, room, dtype=torch.uint8, device=device)
    cache = pkg.Kv4Cache(*(one.as_strided((B, NKV, cap, n), (NKV * room, room, n, 1), p)
                           for p, n in zip(at, (D // 2, D // 2, D // 32, D // 32))))
    plain = pkg.kv4_cache(B, NKV, cap, D, device)
    k, v, slots = randn(rng, B, NKV, T, D).to(device), randn(rng, B, NKV, T, D).to(device), ints([3, cap - T], device)
    for c in (cache, plain):
        pkg.kv4_store(k, v, c, slots)
    assert all(torch.equal(a, b) for a, b in zip(cache, plain))
    both = torch.zeros(B, NKV, 2, T, D, dtype=BF16, device=device)
    pkg.kv4_load(cache, slots, T, both[:, :, 0], both[:, :, 1])
    assert all(torch.equal(a, b) for a, b in zip(both.unbind(2), pkg.kv4_load(plain, slots, T)))


def test_kv4_store_of_one_token(device):
    """Keys [B, NKV, 1, D] beside values that are a view of [B, 1, NKV, D], as a rotated key and a projection's value are: the
    step between tokens differs and is not used. Of two tokens it is, and K and V share it."""
    rng = np.random.default_rng(6)
    B, NKV, D, cap = 2, 4, 128, 30
    k, v, slots = randn(rng, B, NKV, 1, D).to(device), randn(rng, B, 1, NKV, D).to(device).transpose(1, 2), ints([3, 29], device)
    k = torch.as_strided(k, k.shape, (NKV * D, D, D, 1))
    v = torch.as_strided(v, v.shape, (NKV * D, D, NKV * D, 1))
    a, b = (pkg.kv4_store(k, x, pkg.kv4_cache(B, NKV, cap, D, device), slots) for x in (v, v.contiguous()))
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and b.v.any()
    two = randn(rng, B, 2, NKV, D).to(device).transpose(1, 2)
    with pytest.raises(RuntimeError):
        pkg.kv4_store(two.contiguous(), two, a, slots)


def test_window_of_one_row(device):
    """One row's caches, whose steps between rows differ."""
    rng = np.random.default_rng(7)
    q, k, v = (randn(rng, *s).to(device) for s in ((1, 4, 128), (1, 2, 50, 128), (1, 2, 50, 128)))
    lens = ints([50], device)
    want = pkg.gqa_window(q, k, v, lens, 0.1, 20)
    assert torch.equal(pkg.gqa_window(q, k, torch.as_strided(v, v.shape, (8, 50 * 128, 128, 1)), lens, 0.1, 20), want)


# ------------------------------------------------------------------------------------------------- eviction

@pytest.mark.parametrize("shape", ["2bhs", "b2hs", "bh2s", "bsh2"])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_views_of_one_tensor(device, shape, in_place):
    """K and V side by side in one tensor, by any of its dims."""
    rng = np.random.default_rng(3)
    B, NKV, cap, D, keep = 2, 3, 90, 64, 40
    if shape == "bsh2":
        kv = randn(rng, B, cap, NKV, 2, D).to(device).permute(3, 0, 2, 1, 4)
    else:
        sizes = dict(b=B, h=NKV, s=cap)
        kv = randn(rng, *(2 if c == "2" else sizes[c] for c in shape), D).to(device).movedim(shape.index("2"), 0)
    k, v = kv[0], kv[1]
    assert k.shape == (B, NKV, cap, D)
    old, weights = kv.clone(), torch.rand(B, NKV, cap, device=device)
    outs = None if in_place else torch.zeros_like(kv).unbind(0)
    index, lens = pkg.kv_evict((k, v), weights, ints([cap, cap - 7], device), keep, sinks=2, recent=5, outs=outs)
    at = index.long()[..., None].expand(-1, -1, -1, D)
    for i, got in enumerate((k, v) if in_place else outs):
        assert torch.equal(got[:, :, :keep], old[i].gather(2, at))
        assert torch.equal(got[:, :, keep:], old[i][:, :, keep:] if in_place else torch.zeros_like(got[:, :, keep:]))
    assert lens.tolist() == [keep, keep]


def test_evict_refuses_weights_among_the_tensors(device):
    """The weights move with the selection; as one of the tensors they would move twice."""
    rng = np.random.default_rng(4)
    k, w, lens = randn(rng, 1, 2, 64, 64).to(device), torch.rand(1, 2, 64, device=device), ints([64], device)
    held, other = w.clone(), torch.zeros_like(w)
    for call in (lambda: pkg.kv_evict((k, w[..., None]), w, lens, 16),
                 lambda: pkg.kv_evict((other[..., None],), w, lens, 16, outs=(held[..., None],), weights_out=other),
                 lambda: pkg.kv_evict((k, w[..., None]), w, lens, 16, outs=(torch.zeros_like(k), other[..., None]))):
        with pytest.raises(RuntimeError):
            call()
    assert torch.equal(w, held)
    # read by the selection and moved to another place, it is a tensor like any other
    index, _ = pkg.kv_evict((w[..., None],), w, lens, 16, outs=(other[..., None],), weights_out=torch.zeros_like(w))
    assert torch.equal(other[..., :16], held.gather(2, index.long())) and torch.equal(w, held)


# ---------------------------------------------------------------------------------------------- workspaces

def test_batches_of_many_sizes_keep_few_workspaces(device):
    """A stream whose batch moves, with more than 512 units: one workspace a kind up to 1024, every result the row's own."""
    from breeze_tts_2_flash_amd import long_cache
    rng = np.random.default_rng(8)
    NKV, G, D, cap, most = 8, 1, 64, 200, 130
    q, k, v = (randn(rng, *s).to(device) for s in ((most, NKV * G, D), (most, NKV, cap, D), (most, NKV, cap, D)))
    w = torch.rand(most, NKV, cap, device=device)
    lens = ints([cap - b % 50 for b in range(most)], device)
    cache = pkg.kv4_store(k, v, pkg.kv4_cache(most, NKV, cap, D, device), ints([0] * most, device))

    def step(B, splits):
        wo = torch.zeros_like(w[:B])
        c = pkg.Kv4Cache(*(t[:B] for t in cache))
        return (pkg.gqa_window(q[:B], k[:B], v[:B], lens[:B], 0.1, 0, num_splits=splits),
                pkg.gqa_decode_kv4(q[:B], c, lens[:B], 0.1, num_splits=splits),
                pkg.gqa_decode_tracked(q[:B], k[:B], v[:B], lens[:B], 0.1, w[:B], weights_out=wo, num_splits=splits), wo)

    want = step(64, 3)  # 512 units
    ref, spread, reach = window_attention(q[:64].float().cpu()[:, :, None], k[:64].float().cpu(), v[:64].float().cpu(),
                                          lens[:64].tolist(), 0.1)
    assert (np.abs(want[0].float().cpu().numpy() - ref[:, 0]) <= attention_bound(ref, spread, reach, 0.1, D)[:, 0]).all()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for B in (65, 100, 128, 66, 127, 64, 130, 90):
            for got, x in zip(step(B, 3), want):
                assert torch.equal(got[:64], x), B
    side.synchronize()
    keys = [key for key in long_cache._WS if key[1] == side.cuda_stream]
    assert len(keys) == 9, keys  # up to 512, 1024 and 2048 units of each kind


# ---------------------------------------------------------------------------------------- torch.compile

@pytest.mark.parametrize("fmt", ["bf16", "kv4"])
def test_compiled_in_place(device, fmt):
    """The default forms, which write what they read, under torch.compile: outputs and the tensors left as in eager."""
    rng = np.random.default_rng(10)
    B, NKV, cap, D, keep = 2, 2, 300, 128, 90
    q, k, v = (randn(rng, *s).to(device) for s in ((B, 2 * NKV, D), (B, NKV, cap, D), (B, NKV, cap, D)))
    state = [k, v, torch.rand(B, NKV, cap, device=device), ints([300, 222], device)]
    if fmt == "kv4":
        state += pkg.kv4_store(k, v, pkg.kv4_cache(B, NKV, cap, D, device), ints([0, 0], device))

    def step(q, k, v, w, lens, *cache):
        out = pkg.gqa_decode_tracked(q, k, v, lens, 0.1, w, decay=0.5)
        index, n = pkg.kv_evict(pkg.Kv4Cache(*cache) if cache else (k, v), w, lens, keep, sinks=3, recent=7)
        more = pkg.gqa_decode_kv4(q, pkg.Kv4Cache(*cache), n, 0.1) if cache else pkg.gqa_window(q, k, v, n, 0.1, 50)
        return out, index, n, more

    def chosen(w, lens):
        return pkg.kv_select(w, lens, keep, sinks=3, weights_out=w, lens=lens)

    for call, first, mutated in ((step, (q,), True), (chosen, (), False)):
        args = state if mutated else state[2:4]
        a, b = [t.clone() for t in args], [t.clone() for t in args]
        want, got = call(*first, *a), torch.compile(call, fullgraph=True)(*first, *b)
        assert all(torch.equal(x, y) for x, y in zip(want, got)) and all(torch.equal(x, y) for x, y in zip(a, b))
        assert not torch.equal(a[0], args[0]) or fmt == "kv4"


# ------------------------------------------------------------------------------------- terms, and workspaces shared

@pytest.mark.parametrize("T,NKV,G,D,n,splits", [(64, 2, 2, 128, 150, 0), (37, 1, 4, 128, 700, 0), (50, 2, 1, 64, 900, 3), (130, 1, 2, 128, 400, 0),
                                                (100, 1, 2, 64, 2000, 5), (16, 8, 2, 128, 3000, 0), (16, 8, 8, 64, 500, 4)])
def test_split_kernel_holds_two_terms(device, T, NKV, G, D, n, splits):
    """Chunks of fewer column tiles than CUs, which the split kernel takes: softmax terms to 2^-17, not to a bf16's 2^-8."""
    rng = np.random.default_rng(T)
    q, k, v = randn(rng, 1, NKV * G, T, D), randn(rng, 1, NKV, n, D), randn(rng, 1, NKV, n, D)
    out = pkg.gqa_window(q.to(device), k.to(device), v.to(device), ints([n], device), D ** -0.5, 90, sinks=3, num_splits=splits)
    ref, spread, reach = window_attention(q.float(), k.float(), v.float(), [n], D ** -0.5, 90, 3)
    assert (np.abs(out.float().cpu().numpy() - ref) <= attention_bound(ref, spread, reach, D ** -0.5, D)).all()


def test_chunk_splits_share_a_workspace_with_counters(device):
    """A chunk's splits and decode steps in turn in one workspace: the chunk's sums leave the counters at zero."""
    rng = np.random.default_rng(11)
    NKV, G, D, n, T = 8, 2, 128, 5000, 128
    q, k, v = (randn(rng, *s).to(device) for s in ((1, NKV * G, T, D), (1, NKV, n, D), (1, NKV, n, D)))
    lens, row = ints([n], device), q[:, :, -1].contiguous()
    chunk = pkg.long_workspace("window", torch.device("cuda", 0), 1, NKV * G, NKV, D, n, T)
    step = pkg.long_workspace("window", torch.device("cuda", 0), 1, NKV * G, NKV, D, n, 1, num_splits=9)
    assert chunk.numel() > step.numel() > 0
    w = torch.zeros(1, NKV, n, device=device)
    calls = [lambda ws: pkg.gqa_window(q, k, v, lens, D ** -0.5, 0, workspace=ws),
             lambda ws: pkg.gqa_window(row, k, v, lens, D ** -0.5, 0, num_splits=9, workspace=ws),
             lambda ws: pkg.gqa_decode_tracked(row, k, v, lens, D ** -0.5, w, weights_out=torch.zeros_like(w), workspace=ws)]
    want = [f(None) for f in calls]
    for i in (0, 1, 0, 2, 1, 0, 2, 0, 1):
        assert torch.equal(calls[i](chunk), want[i]), i
    last = window_attention(q[:, :, -1:].float().cpu(), k.float().cpu(), v.float().cpu(), [n], D ** -0.5)
    excess = np.abs(want[1].float().cpu().numpy() - last[0][:, 0]) - attention_bound(*last, D ** -0.5, D)[:, 0]
    assert excess.max() <= 0
    excess = np.abs(want[0][:, -1].float().cpu().numpy() - last[0][:, 0]) - attention_bound(*last, D ** -0.5, D, True)[:, 0]
    assert excess.max() <= 0


def test_longest_chunk(device):
    """The chunk kernel's grid holds 65535 column tiles: 65535 * 16 tokens of 8 q heads; longer ones are refused, not launched."""
    dev, size = torch.device("cuda", 0), (1, 8, 1, 64, 1 << 22)
    assert pkg.long_workspace("window", dev, *size, 65535 * 16, num_splits=1).numel() == 0
    with pytest.raises(RuntimeError):
        pkg.long_workspace("window", dev, *size, 65535 * 16 + 1, num_splits=1)
    q = torch.zeros(1, 8, 1, 64, dtype=BF16, device=device).expand(1, 8, 1 << 20, 64)
    k = torch.zeros(1, 1, 64, 64, dtype=BF16, device=device)
    with pytest.raises(RuntimeError):
        pkg.gqa_window(q, k, k, ints([64], device), 0.1, 0, torch.empty(1, 1 << 20, 8, 64, dtype=BF16, device=device), num_splits=1)


def test_chunks_captured_and_replayed(device):
    """A chunk in splits, one whole, a window's and the 4-bit calls in one graph, on lengths and inputs that change between the
    replays, with eager work between them; every replay as in eager."""
    rng = np.random.default_rng(12)
    dev, NKV, G, D, n = torch.device("cuda", 0), 8, 2, 128, 4000
    q, k, v = (randn(rng, *s).to(device) for s in ((1, NKV * G, 400, D), (1, NKV, n, D), (1, NKV, n, D)))
    few = q[:, :, :128].contiguous()
    lens, slot, cache = ints([n], device), ints([0], device), pkg.kv4_cache(1, NKV, 64, D, device)
    ws = pkg.long_workspace("window", dev, 1, NKV * G, NKV, D, n, 128)
    assert ws.numel() > 0 and pkg.long_workspace("window", dev, 1, NKV * G, NKV, D, n, 400, window=90).numel() == 0

    def run(ws):
        pkg.kv4_store(k[:, :, :64], v[:, :, :64], cache, slot)
        return [pkg.gqa_window(few, k, v, lens, D ** -0.5, 0, workspace=ws), pkg.gqa_window(q, k, v, lens, D ** -0.5, 90, sinks=3),
                *pkg.kv4_load(cache, slot, 50)]

    run(ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(ws)
    for i in range(4):
        lens.fill_(n - 777 * i)
        slot.fill_(i)
        q.copy_(randn(rng, *q.shape))
        few.copy_(q[:, :, 100:228])
        graph.replay()
        torch.cuda.synchronize()
        held = [t.clone() for t in got]
        for a, b in zip(held, run(None)):
            assert torch.equal(a, b), i
