"""GPU: the long-cache operators (include/bz_long_cache.h) against their float64 oracles: sliding-window attention with sinks,
the 4-bit cache, accumulated attention weights, selection and compaction. Tolerances are oracle.long_cache.attention_bound's
(derived there); codes, scales, moved rows and choices are compared exactly."""
import numpy as np
import pytest
import torch

import breeze_tts_2_flash_amd as pkg
from oracle.long_cache import attention_bound, kv4_round, select, window_attention

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def ints(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def randn(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(BF16)


def check_attention(out, q, k, v, lens, scale, window=0, sinks=0, starts=None, what=""):
    """out [B, T, NH, D] of q [B, NH, T, D] (CPU tensors or arrays)."""
    D = q.shape[-1]
    ref, spread, reach = window_attention(q, k, v, lens, scale, window, sinks, starts)
    got = out.float().cpu().numpy().astype(np.float64).reshape(ref.shape)
    one_term = q.shape[2] * q.shape[1] // k.shape[1] >= 64  # a chunk: 64 (token, q head) pairs of a kv head or more
    excess = np.abs(got - ref) - attention_bound(ref, spread, reach, scale, D, one_term)
    assert np.isfinite(got).all(), f"{what}: non-finite"
    assert excess.max() <= 0, f"{what}: {excess.max():.3e} past the bound at {np.unravel_index(excess.argmax(), excess.shape)}"
    return ref


def poison(k, v, lens, starts, T, window, sinks, value=float("nan")):
    """k, v with `value` wherever no token of the row looks."""
    from oracle.long_cache import attended
    k, v = k.clone(), v.clone()
    for b in range(k.size(0)):
        e = min(max(lens[b], 0), k.size(2))
        s = min(max(starts[b], 0), e) if starts is not None else 0
        seen = set().union(*map(set, attended(s, e, T, window, sinks)))
        out = [p for p in range(k.size(2)) if p not in seen]
        k[b, :, out] = value
        v[b, :, out] = value
    return k, v


WINDOW_CASES = [
    # NKV, G, D, cap, T, lens, starts, window, sinks
    (2, 1, 128, 70, 1, [70, 1, 0, 33], None, 16, 4),
    (2, 2, 128, 300, 1, [300, 257, 16, 5], [0, 40, 3, 5], 100, 4),
    (1, 4, 64, 520, 1, [520, 300], [7, 0], 1, 0),
    (1, 8, 128, 200, 1, [200, 199], None, 0, 0),
    (2, 2, 64, 333, 1, [333, 100], [0, 99], 64, 33),
    (2, 2, 128, 150, 3, [150, 2, 0], [0, 0, 0], 32, 5),
    (1, 8, 64, 100, 2, [99, 100], [50, 0], 17, 1),
    (1, 4, 128, 140, 37, [140, 37, 12], [3, 0, 0], 20, 2),
    (2, 1, 64, 90, 50, [90, 60], None, 0, 0),
    (1, 2, 128, 400, 130, [400, 130, 131], [0, 10, 0], 48, 7),
    (1, 2, 64, 64, 64, [64], None, 1000, 1000),
    (1, 2, 128, 260, 257, [257, 260], [0, 100], 70, 0),
    (1, 1, 128, 200, 200, [200], None, 129, 3),
    # as many columns as the chunk kernel takes, by one, two and four column groups of a workgroup
    (8, 4, 128, 200, 160, [200, 170], [30, 0], 77, 4),
    (8, 8, 64, 150, 150, [150, 149, 3], [0, 5, 0], 40, 9),
    (8, 8, 128, 330, 300, [330, 300], None, 100, 0),
    (8, 8, 64, 515, 515, [515, 400, 90], [0, 3, 0], 0, 0),
    (8, 8, 128, 390, 390, [390, 389, 200, 1], [0, 30, 0, 0], 64, 1),
]


@pytest.mark.parametrize("case", WINDOW_CASES, ids=lambda c: f"kv{c[0]}g{c[1]}d{c[2]}T{c[4]}w{c[7]}s{c[8]}")
def test_window_against_oracle(device, case):
    NKV, G, D, cap, T, lens, starts, window, sinks = case
    rng = np.random.default_rng(cap + T)
    B = len(lens)
    q, k, v = randn(rng, B, NKV * G, T, D), randn(rng, B, NKV, cap, D), randn(rng, B, NKV, cap, D)
    k[:, :, :: 17] *= 4
    kp, vp = poison(k, v, lens, starts, T, window, sinks)
    out = pkg.gqa_window(q.to(device), kp.to(device), vp.to(device), ints(lens, device), D ** -0.5, window, sinks=sinks,
                         kv_start=None if starts is None else ints(starts, device))
    torch.cuda.synchronize()
    assert tuple(out.shape) == ((B, NKV * G, D) if T == 1 else (B, T, NKV * G, D))
    ref = check_attention(out, q.float(), k.float(), v.float(), lens, D ** -0.5, window, sinks, starts)
    assert (out.float().cpu().numpy().reshape(ref.shape)[ref == 0] == 0).all()  # rows that attend nothing


@pytest.mark.parametrize("splits", [0, 1, 2, 5, 64, 256])
@pytest.mark.parametrize("kind", ["window", "kv4"])
def test_long_rows_and_split_counts(device, kind, splits):
    rng = np.random.default_rng(splits)
    B, NKV, G, D, cap, T = 2, 2, 2, 128, 3000, 2
    lens, starts, window, sinks = [3000, 2111], [0, 100], 1500, 70
    q, k, v = randn(rng, B, NKV * G, T, D), randn(rng, B, NKV, cap, D), randn(rng, B, NKV, cap, D)
    args = dict(kv_start=ints(starts, device), sinks=sinks, num_splits=splits)
    if kind == "kv4":
        cache = pkg.kv4_store(k.to(device), v.to(device), pkg.kv4_cache(B, NKV, cap, D, device), ints([0, 0], device))
        out = pkg.gqa_decode_kv4(q.to(device), cache, ints(lens, device), D ** -0.5, window=window, **args)
        k, v = kv4_round(k.float().numpy())[0], kv4_round(v.float().numpy())[0]
    else:
        out = pkg.gqa_window(q.to(device), k.to(device), v.to(device), ints(lens, device), D ** -0.5, window, **args)
        k, v = k.float(), v.float()
    torch.cuda.synchronize()
    check_attention(out, q.float(), k, v, lens, D ** -0.5, window, sinks, starts, f"{kind} splits {splits}")


@pytest.mark.parametrize("T", [1, 4, 100])
def test_window_layouts(device, T):
    """Strided q and out, a [B, capacity, NKV, D] cache, int32 tensors in the middle of others."""
    rng = np.random.default_rng(T)
    B, NKV, G, D, cap = 2, 2, 2, 64, 150
    q, k, v = randn(rng, B, NKV * G, T, D), randn(rng, B, NKV, cap, D), randn(rng, B, NKV, cap, D)
    lens, starts = [150, 120], [0, 9]
    kv = torch.stack([k, v], 3).permute(0, 2, 1, 3, 4).contiguous().to(device)  # [B, cap, NKV, 2, D]
    kd, vd = kv[:, :, :, 0].permute(0, 2, 1, 3), kv[:, :, :, 1].permute(0, 2, 1, 3)
    wide = torch.zeros(B, T, NKV * G, D + 8, dtype=BF16, device=device)
    wide[..., :D] = q.transpose(1, 2)
    qd = wide[..., :D].transpose(1, 2)
    full = torch.full((B, NKV * G, T, D + 8), 7.0, dtype=BF16, device=device)
    pkg.gqa_window(qd, kd, vd, ints([0] + lens, device)[1:], D ** -0.5, 40, full[..., :D], sinks=3,
                   kv_start=ints([0] + starts, device)[1:])
    torch.cuda.synchronize()
    # where T == NH the shape is read as [B, T, NH, D], the reference's layout
    out = full[..., :D] if T == NKV * G else full[..., :D].transpose(1, 2)
    check_attention(out, q.float(), k.float(), v.float(), lens, D ** -0.5, 40, 3, starts)
    assert (full[..., D:] == 7).all()


@pytest.mark.parametrize("splits", [2, 3, 7, 40])
@pytest.mark.parametrize("NKV,G,D,cap,T,lens,starts,window,sinks", [
    (8, 4, 128, 1300, 160, [1300, 700], [30, 0], 0, 0), (8, 8, 64, 900, 150, [900, 149, 3], [0, 5, 0], 300, 70),
    (8, 2, 128, 2000, 333, [2000, 333, 0], None, 700, 4), (16, 1, 64, 1500, 260, [1500], [99], 0, 3),
])
def test_chunk_splits(device, NKV, G, D, cap, T, lens, starts, window, sinks, splits):
    """A chunk whose positions are shared out to workgroups; rows that are shorter than the chunk, or empty."""
    rng = np.random.default_rng(T + splits)
    B = len(lens)
    q, k, v = randn(rng, B, NKV * G, T, D), randn(rng, B, NKV, cap, D), randn(rng, B, NKV, cap, D)
    k[:, :, :: 17] *= 4
    kp, vp = poison(k, v, lens, starts, T, window, sinks)
    out = pkg.gqa_window(q.to(device), kp.to(device), vp.to(device), ints(lens, device), D ** -0.5, window, sinks=sinks,
                         kv_start=None if starts is None else ints(starts, device), num_splits=splits)
    ref = check_attention(out, q.float(), k.float(), v.float(), lens, D ** -0.5, window, sinks, starts)
    assert (out.float().cpu().numpy().reshape(ref.shape)[ref == 0] == 0).all()  # rows that attend nothing


@pytest.mark.parametrize("T,G,D,n,window", [(128, 2, 128, 5000, 0), (200, 2, 64, 4500, 0), (70, 4, 128, 4200, 4000)])
def test_chunk_behind_a_long_context(device, T, G, D, n, window):
    """Few tokens over many positions, whose splits the library chooses; the same with a workspace of the caller's."""
    rng = np.random.default_rng(T)
    NKV = 8
    q, k, v = randn(rng, 1, NKV * G, T, D), randn(rng, 1, NKV, n + 9, D), randn(rng, 1, NKV, n + 9, D)
    k[:, :, n:], v[:, :, n:] = float("nan"), float("nan")
    args = (q.to(device), k.to(device), v.to(device), ints([n], device), D ** -0.5, window)
    out = pkg.gqa_window(*args, sinks=2)
    check_attention(out, q.float(), k[:, :, :n].float(), v[:, :, :n].float(), [n], D ** -0.5, window, 2)
    ws = pkg.long_workspace("window", torch.device("cuda", 0), 1, NKV * G, NKV, D, n + 9, T, window=window, sinks=2)
    assert ws.numel() > 0
    for _ in range(2):
        assert torch.equal(pkg.gqa_window(*args, sinks=2, workspace=ws), out)
    with pytest.raises(RuntimeError):
        pkg.gqa_window(*args, sinks=2, workspace=ws[:-256])


# the split kernel, and the chunk kernel by one, two and four column groups, and split
@pytest.mark.parametrize("T,NKV,G,D", [(3, 1, 2, 128), (70, 1, 2, 128), (70, 8, 8, 128), (70, 8, 8, 64), (130, 32, 8, 128),
                                       (800, 64, 2, 128), (800, 64, 2, 64)])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("splits", [0, 3])
def test_unattended_values_do_not_reach_a_token(device, T, NKV, G, D, value, splits):
    """A position that some tokens of a chunk attend and others do not: only those that do may see what it holds."""
    rng = np.random.default_rng(T)
    n, window, sinks = T + 130, 30, 2
    q, k, v = randn(rng, 1, NKV * G, T, D), randn(rng, 1, NKV, n, D), randn(rng, 1, NKV, n, D)
    at = [n - 1, n - T + 1, n - T - window + 2]
    vp = v.clone()
    vp[0, 0, at, 5] = value
    out = pkg.gqa_window(q.to(device), k.to(device), vp.to(device), ints([n], device), D ** -0.5, window, sinks=sinks, num_splits=splits)
    assert torch.isfinite(out[0, :, G:].float()).all()  # the other kv heads
    out = out.float().cpu()[0, :, :G]
    clean = pkg.gqa_window(q.to(device), k.to(device), v.to(device), ints([n], device), D ** -0.5, window, sinks=sinks, num_splits=splits)
    clean = clean.float().cpu()[0, :, :G]
    from oracle.long_cache import attended
    for t, pos in enumerate(attended(0, n, T, window, sinks)):
        hit = any(a in pos for a in at)
        rest = [d for d in range(D) if d != 5]
        assert torch.isfinite(out[t][:, rest]).all(), t
        assert (out[t][:, rest] - clean[t][:, rest]).abs().max() <= 2.0 ** -7 * clean[t].abs().max(), t
        if not hit:
            assert torch.isfinite(out[t]).all(), t
        elif value != value:
            assert torch.isnan(out[t][:, 5]).all(), t
        else:
            assert (out[t][:, 5] == value).all(), (t, out[t][:, 5])
    # keys: a NaN key poisons exactly the tokens that attend it
    kp = k.clone()
    kp[0, 0, n - 1] = float("nan")
    out = pkg.gqa_window(q.to(device), kp.to(device), v.to(device), ints([n], device), D ** -0.5, window, sinks=sinks, num_splits=splits)
    assert torch.isnan(out[0, T - 1, :G].float()).all() and torch.isfinite(out[0, :T - 1].float()).all()


@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
@pytest.mark.parametrize("T", [1, 64])
def test_scales(device, T, scale):
    """A negative scale, none, and one that leaves a single position."""
    rng = np.random.default_rng(T)
    NKV, G, D, n = 2, 2, 128, 150
    q, k, v = randn(rng, 1, NKV * G, T, D), randn(rng, 1, NKV, n, D), randn(rng, 1, NKV, n, D)
    out = pkg.gqa_window(q.to(device), k.to(device), v.to(device), ints([n], device), scale, 60, sinks=3)
    check_attention(out, q.float(), k.float(), v.float(), [n], scale, 60, 3)
    if T == 1:
        cache = pkg.kv4_store(k.to(device), v.to(device), pkg.kv4_cache(1, NKV, n, D, device), ints([0], device))
        out = pkg.gqa_decode_kv4(q.to(device), cache, ints([n], device), scale)
        check_attention(out, q.float(), kv4_round(k.float().numpy())[0], kv4_round(v.float().numpy())[0], [n], scale)


def test_window_equals_plain_decode(device):
    """Without a window it is gqa_decode's attention."""
    rng = np.random.default_rng(5)
    B, NKV, G, D, cap = 3, 8, 2, 128, 700
    q, k, v = (x.to(device) for x in (randn(rng, B, NKV * G, D), randn(rng, B, NKV, cap, D), randn(rng, B, NKV, cap, D)))
    lens, starts = ints([700, 512, 31], device), ints([0, 20, 0], device)
    a = pkg.gqa_window(q, k, v, lens, D ** -0.5, 0, kv_start=starts).float()
    b = pkg.gqa_decode(q, k, v, lens, D ** -0.5, kv_start=starts).float()
    assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 1e-5).all()


# --------------------------------------------------------------------------------------------------- 4 bits

def special_values(rng, shape):
    x = randn(rng, *shape).float().numpy()
    x = x * np.exp2(rng.integers(-12, 12, (*shape[:-1], 1)))
    x[..., 0, :] = 0
    x[..., 1, :32] *= 2.0 ** -130  # subnormal blocks
    x[..., 2, 33] = 3e38
    return torch.from_numpy(x.astype(np.float32)).to(BF16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [3, 40])
def test_kv4_store_load(device, D, T):
    rng = np.random.default_rng(D + T)
    B, NKV, cap = 3, 2, 61
    k, v = special_values(rng, (B, NKV, T, D)), special_values(rng, (B, NKV, T, D))
    k[1, 0, 2, 40] = float("inf")
    v[1, 1, 1, 5] = float("nan")
    slots, counts = [0, 30, -2], [T, 2, T]
    cache = pkg.kv4_cache(B, NKV, cap, D, device)
    for t in cache:
        t.fill_(0xA5)
    before = [t.cpu().numpy().copy() for t in cache]
    pkg.kv4_store(k.to(device), v.to(device), cache, ints(slots, device), counts=ints(counts, device))
    lk, lv = pkg.kv4_load(cache, ints(slots, device), T)
    torch.cuda.synchronize()
    for x, codes, scales, got, i in ((k, 0, 2, lk, 0), (v, 1, 3, lv, 1)):
        values, c, E = kv4_round(x.float().numpy())
        want_c, want_e = before[codes].copy(), before[scales].copy()
        for b in range(B):
            for t in range(T):
                p = slots[b] + t
                if t < counts[b] and 0 <= p < cap:
                    want_c[b, :, p], want_e[b, :, p] = c[b, :, t], E[b, :, t]
                    assert np.array_equal(got[b, :, t].float().cpu().numpy(), values[b, :, t].astype(np.float32), equal_nan=True)
                elif not 0 <= p < cap:
                    assert (got[b, :, t] == 0).all()
        assert np.array_equal(cache[codes].cpu().numpy(), want_c)
        assert np.array_equal(cache[scales].cpu().numpy(), want_e)


def test_kv4_every_bf16_value(device):
    """Every finite bf16 value as the largest of its block, beside ties of its scale (and blocks that overflow)."""
    bits = np.arange(0, 0x7F80, dtype=np.uint32)
    big = (bits << 16).view(np.float32)
    x = np.zeros((len(big), 64), np.float32)
    x[:, 0] = big
    with np.errstate(over="ignore", under="ignore"):
        for i, f in enumerate([0.25, 0.5, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0]):
            x[:, 1 + i] = big * np.float32(f / 7)
            x[:, 32 + i] = -big * np.float32(f / 4)
    x = torch.from_numpy(x).to(BF16)[None, None]
    n = x.size(2)
    cache = pkg.kv4_cache(1, 1, n, 64, device)
    pkg.kv4_store(x.to(device), x.to(device), cache, ints([0], device))
    got, _ = pkg.kv4_load(cache, ints([0], device), n)
    values, codes, E = kv4_round(x.float().numpy())
    assert np.array_equal(cache.k.cpu().numpy(), codes) and np.array_equal(cache.v_scale.cpu().numpy(), E)
    with np.errstate(over="ignore"):  # blocks past the largest bf16 are infinite or NaN on both sides
        assert np.array_equal(got.float().cpu().numpy(), values.astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("NKV,G,D,cap,T,lens,starts,window,sinks", [
    (2, 1, 128, 70, 1, [70, 1, 0, 33], None, 0, 0),
    (2, 2, 128, 301, 1, [301, 257, 16, 5], [0, 40, 3, 5], 100, 4),
    (1, 4, 64, 521, 1, [521, 300], [7, 0], 0, 0),
    (1, 8, 128, 200, 2, [200, 199], None, 0, 0),
    (2, 2, 64, 333, 5, [333, 100, 3], [0, 99, 0], 64, 33),
    (1, 8, 64, 99, 16, [99, 40], [50, 0], 17, 1),
    (1, 1, 128, 140, 16, [140, 12], None, 33, 2),
])
def test_kv4_attention(device, NKV, G, D, cap, T, lens, starts, window, sinks):
    rng = np.random.default_rng(cap)
    B = len(lens)
    q, k, v = randn(rng, B, NKV * G, T, D), randn(rng, B, NKV, cap, D), randn(rng, B, NKV, cap, D)
    kp, vp = poison(k, v, lens, starts, T, window, sinks)
    cache = pkg.kv4_store(kp.to(device), vp.to(device), pkg.kv4_cache(B, NKV, cap, D, device), ints([0] * B, device))
    out = pkg.gqa_decode_kv4(q.to(device), cache, ints(lens, device), D ** -0.5,
                             kv_start=None if starts is None else ints(starts, device), window=window, sinks=sinks)
    torch.cuda.synchronize()
    check_attention(out, q.float(), kv4_round(k.float().numpy())[0], kv4_round(v.float().numpy())[0], lens, D ** -0.5, window,
                    sinks, starts)


@pytest.mark.parametrize("D", [64, 128])
def test_kv4_strided_cache(device, D):
    """Codes [B, capacity, NKV, D / 2] with K and V side by side, scales in views: the same cache otherwise."""
    rng = np.random.default_rng(D)
    B, NKV, G, cap = 2, 2, 2, 150
    codes = torch.zeros(B, cap, NKV, 2, D // 2, dtype=torch.uint8, device=device).permute(0, 2, 1, 3, 4)
    scales = torch.zeros(B, NKV + 1, 2, cap + 6, D // 32, dtype=torch.uint8, device=device)
    cache = pkg.Kv4Cache(codes[:, :, :, 0], codes[:, :, :, 1], scales[:, 1:, 0, 2:cap + 2], scales[:, 1:, 1, 2:cap + 2])
    plain = pkg.kv4_cache(B, NKV, cap, D, device)
    q, k, v = randn(rng, B, NKV * G, D).to(device), randn(rng, B, NKV, cap, D).to(device), randn(rng, B, NKV, cap, D).to(device)
    zero, lens = ints([0, 0], device), ints([150, 77], device)
    for c in (cache, plain):
        pkg.kv4_store(k, v, c, zero)
    assert all(torch.equal(a, b) for a, b in zip(cache, plain))
    assert all(torch.equal(a, b) for a, b in zip(pkg.kv4_load(cache, zero, cap), pkg.kv4_load(plain, zero, cap)))
    a, b = (pkg.gqa_decode_kv4(q, c, lens, D ** -0.5, window=100, sinks=3) for c in (cache, plain))
    assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_kv4_values_past_bf16(device, D, sign):
    """A block whose largest value is above 1.75 2^127 loads it as an infinity (4 times 2^126): it reaches the tokens that
    attend its position, and no other of the tile."""
    rng = np.random.default_rng(D)
    T, n, at = 4, 40, 30  # window 8: tokens 0 and 1 attend position 30, 2 and 3 do not
    q, k, v = randn(rng, 1, 2, T, D), randn(rng, 1, 1, 64, D), randn(rng, 1, 1, 64, D)
    v[0, 0, at, 7] = sign * 3.38e38
    cache = pkg.kv4_store(k.to(device), v.to(device), pkg.kv4_cache(1, 1, 64, D, device), ints([0], device))
    lk, lv = (x.float().cpu() for x in pkg.kv4_load(cache, ints([0], device), 64))
    assert lv[0, 0, at, 7] == sign * float("inf")
    out = pkg.gqa_decode_kv4(q.to(device), cache, ints([n], device), D ** -0.5, window=8).float().cpu()
    assert (out[0, :2, :, 7] == sign * float("inf")).all()
    rest = lv.clone()
    rest[0, 0, at] = 0
    ref, spread, reach = window_attention(q.float(), lk, rest, [n], D ** -0.5, 8, 0, None)
    excess = np.abs(out.numpy() - ref) - attention_bound(ref, spread, reach, D ** -0.5, D, False)
    assert np.isfinite(out[0, 2:].numpy()).all() and excess[0, 2:].max() <= 0


def test_kv4_attention_reads_what_load_returns(device):
    """The attention over the codes is the window attention over kv4_load's values, to the last bf16 step."""
    rng = np.random.default_rng(3)
    B, NKV, G, D, cap, T = 2, 2, 4, 128, 500, 3
    q, k, v = (x.to(device) for x in (randn(rng, B, NKV * G, T, D), randn(rng, B, NKV, cap, D), randn(rng, B, NKV, cap, D)))
    lens = ints([500, 333], device)
    cache = pkg.kv4_store(k, v, pkg.kv4_cache(B, NKV, cap, D, device), ints([0, 0], device))
    lk, lv = pkg.kv4_load(cache, ints([0, 0], device), cap)
    a = pkg.gqa_decode_kv4(q, cache, lens, D ** -0.5, window=200, sinks=4).float()
    b = pkg.gqa_window(q, lk, lv, lens, D ** -0.5, 200, sinks=4).float()
    assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 1e-5).all()


# ------------------------------------------------------------------------------------------------- eviction

@pytest.mark.parametrize("NKV,G,D,cap,lens,starts", [
    (2, 1, 64, 77, [77, 1, 0], None), (2, 2, 128, 300, [300, 250], [0, 33]), (1, 4, 128, 1500, [1500, 1023], [1, 0]),
    (1, 8, 64, 2050, [2050], None),
])
@pytest.mark.parametrize("decay,in_place", [(1.0, True), (0.5, False), (0.0, False)])
def test_tracked(device, NKV, G, D, cap, lens, starts, decay, in_place):
    rng = np.random.default_rng(cap)
    B = len(lens)
    q, k, v = randn(rng, B, NKV * G, D), randn(rng, B, NKV, cap, D), randn(rng, B, NKV, cap, D)
    kp, vp = poison(k, v, lens, starts, 1, 0, 0)
    w0 = torch.rand(B, NKV, cap, generator=torch.Generator().manual_seed(1))
    w = w0.to(device)
    if decay == 0:
        w.fill_(float("nan"))  # not read
    wo = w if in_place else torch.full_like(w, -3.0)
    out = pkg.gqa_decode_tracked(q.to(device), kp.to(device), vp.to(device), ints(lens, device), D ** -0.5, w, decay=decay,
                                 weights_out=None if in_place else wo, kv_start=None if starts is None else ints(starts, device))
    torch.cuda.synchronize()
    check_attention(out, q.float()[:, :, None], k.float(), v.float(), lens, D ** -0.5, 0, 0, starts)
    # a probability is off by the relative bound of attention_bound's terms
    _, _, reach = window_attention(q.float()[:, :, None], k.float(), v.float(), lens, D ** -0.5, kv_start=starts)
    want = np.full((B, NKV, cap), -3.0) if not in_place else w0.numpy().astype(np.float64)
    tol = np.zeros((B, NKV, cap))
    for b in range(B):
        s, e = (starts[b] if starts else 0), lens[b]
        for h in range(NKV):
            p = np.zeros(e - s)
            for g in range(G):
                x = k[b, h, s:e].double().numpy() @ q[b, h * G + g].double().numpy() * D ** -0.5
                x = np.exp(x - x.max(initial=-np.inf))
                p += x / max(x.sum(), 1e-300)
            want[b, h, s:e] = decay * w0[b, h, s:e].double().numpy() + p
            eps = 4 * D ** -0.5 * reach[b, 0, h * G:(h + 1) * G].max() * (D + 2) * 2.0 ** -23 + 2.0 ** -19
            tol[b, h, s:e] = eps * p + 2.0 ** -23 * want[b, h, s:e]
    assert (np.abs(wo.cpu().numpy() - want) <= tol).all()


def heavy(rng, shape):
    """Accumulated weights with many ties, both zeros, infinities, negatives and NaN."""
    w = np.floor(np.exp(rng.standard_normal(shape)) * 8) / 8
    flat = w.reshape(-1)
    flat[rng.integers(0, flat.size, 5)] = np.nan
    flat[rng.integers(0, flat.size, 3)] = np.inf
    flat[rng.integers(0, flat.size, 9)] = -0.0
    flat[rng.integers(0, flat.size, 9)] *= -1
    return w.astype(np.float32)


@pytest.mark.parametrize("cap,lens,starts,keep,sinks,recent", [
    (50, [50, 7, 0], None, 20, 2, 5), (300, [300, 250, 64], [0, 33, 0], 64, 4, 60), (2100, [2100, 1030], [5, 0], 1024, 0, 0),
    (5000, [5000, 4097], None, 1, 0, 0), (1111, [1111], None, 1110, 3, 100), (700, [700, 400], [0, 1], 399, 0, 399),
    (9000, [9000], None, 4000, 8, 128), (64, [64], None, 64, 1, 1), (70000, [70000, 40001], [0, 3], 33000, 4, 100), (40000, [39999], None, 20000, 0, 0),
])
def test_select(device, cap, lens, starts, keep, sinks, recent):
    rng = np.random.default_rng(cap)
    B, NKV = len(lens), 3
    w = heavy(rng, (B, NKV, cap))
    index, kept, moved = select(w, lens, keep, sinks, recent, starts)
    wd = torch.from_numpy(w).to(device)
    st = None if starts is None else ints(starts, device)
    got, n = pkg.kv_select(wd, ints(lens, device), keep, sinks=sinks, recent=recent, kv_start=st)
    torch.cuda.synchronize()
    assert np.array_equal(got.cpu().numpy(), index) and np.array_equal(n.cpu().numpy(), kept)
    assert np.array_equal(wd.cpu().numpy(), w, equal_nan=True)
    wo = torch.full_like(wd, -5.0)
    pkg.kv_select(wd, ints(lens, device), keep, sinks=sinks, recent=recent, kv_start=st, weights_out=wo)
    for b in range(B):
        assert np.array_equal(wo[b, :, :lens[b]].cpu().numpy(), moved[b, :, :lens[b]], equal_nan=True)
        assert (wo[b, :, lens[b]:] == -5).all()
    ld = ints(lens, device)
    pkg.kv_select(wd, ld, keep, sinks=sinks, recent=recent, kv_start=st, weights_out=wd, lens=ld)  # all in place
    assert np.array_equal(wd.cpu().numpy(), moved, equal_nan=True) and np.array_equal(ld.cpu().numpy(), kept)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("cap,lens,keep", [(50, [50, 7, 0], 20), (2000, [2000, 1500], 1200), (700, [700], 699)])
def test_compact(device, in_place, cap, lens, keep):
    rng = np.random.default_rng(cap)
    B, NKV = len(lens), 2
    index, kept, _ = select(heavy(rng, (B, NKV, cap)), lens, keep, 2, 3)
    tensors = [torch.randint(0, 255, (B, NKV, cap, w), dtype=torch.uint8, device=device) for w in (64, 64, 4, 3)]
    tensors[0] = randn(rng, B, NKV, cap, 72).to(device)[..., 4:68]  # bf16 rows 8 bytes off a 16-byte boundary
    before = [t.cpu().clone() for t in tensors]
    outs = None if in_place else [torch.zeros_like(t) for t in tensors]
    res = pkg.kv_compact(tensors, torch.from_numpy(index).to(device), ints(kept.tolist(), device), outs)
    torch.cuda.synchronize()
    for t, r, old in zip(tensors, res, before):
        want = old.clone() if in_place else torch.zeros_like(old)
        for b in range(B):
            for h in range(NKV):
                want[b, h, :kept[b]] = old[b, h, torch.from_numpy(index[b, h, :kept[b]].astype(np.int64))]
        assert torch.equal(r.cpu(), want)
        if not in_place:
            assert torch.equal(t.cpu(), old)


def test_compact_some_in_place(device):
    """Some tensors of a call move in place and some do not; more rows than a step of either holds."""
    rng = np.random.default_rng(8)
    cap, keep = 9000, 4000
    index, kept, _ = select(heavy(rng, (1, 2, cap)), [cap], keep, 2, 3)
    a, b, c = (torch.randint(0, 255, (1, 2, cap, w), dtype=torch.uint8, device=device) for w in (256, 96, 4))
    old, out = [t.clone() for t in (a, b, c)], torch.zeros_like(b)
    pkg.kv_compact((a, b, c), torch.from_numpy(index).to(device), ints(kept.tolist(), device), (a, out, c))
    at = torch.from_numpy(index.astype(np.int64)).to(device)[..., None]
    for got, t in ((a, old[0]), (out, old[1]), (c, old[2])):
        assert torch.equal(got[:, :, :keep], t.gather(2, at.expand(-1, -1, -1, t.size(3))))
    assert torch.equal(a[:, :, keep:], old[0][:, :, keep:]) and torch.equal(b, old[1]) and (out[:, :, keep:] == 0).all()


def test_compact_leaves_bad_indices_alone(device):
    t = torch.arange(8, device=device, dtype=torch.int64).view(1, 1, 8, 1)
    out = torch.full_like(t, -1)
    index = ints([[[3, -1, 8, 2**31 - 1, 7, 0]]], device)
    pkg.kv_compact((t,), index, ints([5], device), (out,))
    assert out.flatten().tolist() == [3, -1, -1, -1, 7, -1, -1, -1]


def test_compact_interleaved_views_and_overlaps(device):
    kv = torch.arange(2 * 10 * 2 * 8, device=device, dtype=torch.int32).view(1, 10, 2, 2, 8)  # [B, cap, NKV, 2, X]
    k, v = kv[:, :, :, 0].permute(0, 2, 1, 3), kv[:, :, :, 1].permute(0, 2, 1, 3)
    old = kv.clone()
    index = ints([[[0, 4, 9], [1, 2, 5]]], device)
    pkg.kv_compact((k, v), index, ints([3], device))
    for h in range(2):
        for d, i in enumerate(index[0, h].tolist()):
            assert torch.equal(kv[0, d, h], old[0, i, h])
    x = torch.zeros(1, 2, 10, 8, device=device)
    with pytest.raises(RuntimeError):
        pkg.kv_compact((x, x), index, ints([3], device))
    with pytest.raises(RuntimeError):
        pkg.kv_compact((x[:, :, :9],), index, ints([3], device), (x[:, :, 1:],))
    with pytest.raises(RuntimeError):
        pkg.kv_compact((x,), index, ints([3], device), (x[:, :1].expand(1, 2, 10, 8),))


# ---------------------------------------------------------------------------------------- together, streams, graphs

@pytest.mark.parametrize("fmt", ["bf16", "kv4"])
def test_bounded_generation(device, fmt):
    """A cache kept to a budget, as a serving loop does it: a prompt through gqa_window, decode steps that append and
    accumulate weights, an eviction when the cache is full, and steps over what stayed; every output against the oracle on
    the positions that are there."""
    rng = np.random.default_rng(9)
    B, NKV, G, D, cap, prompt, keep = 2, 2, 2, 128, 96, 60, 40
    scale = D ** -0.5
    K, V = torch.zeros(B, NKV, cap, D, dtype=BF16, device=device), torch.zeros(B, NKV, cap, D, dtype=BF16, device=device)
    q, k, v = randn(rng, B, NKV * G, prompt, D), randn(rng, B, NKV, prompt, D), randn(rng, B, NKV, prompt, D)
    K[:, :, :prompt], V[:, :, :prompt] = k.to(device), v.to(device)
    lens = ints([prompt] * B, device)
    out = pkg.gqa_window(q.to(device), K, V, lens, scale, 32, sinks=4)
    check_attention(out, q.float(), k.float(), v.float(), [prompt] * B, scale, 32, 4)
    cache = pkg.kv4_store(K[:, :, :prompt], V[:, :, :prompt], pkg.kv4_cache(B, NKV, cap, D, device), ints([0] * B, device))
    weights = torch.zeros(B, NKV, cap, device=device)
    for step in range(50):
        q, k, v = randn(rng, B, NKV * G, D), randn(rng, B, NKV, 1, D), randn(rng, B, NKV, 1, D)
        n = int(lens[0])
        K[:, :, n], V[:, :, n] = k[:, :, 0].to(device), v[:, :, 0].to(device)
        pkg.kv4_store(k.to(device), v.to(device), cache, lens)
        lens += 1
        out = pkg.gqa_decode_tracked(q.to(device), K, V, lens, scale, weights)
        check_attention(out, q.float()[:, :, None], K.float().cpu(), V.float().cpu(), lens.tolist(), scale, what=f"step {step}")
        out = pkg.gqa_decode_kv4(q.to(device), cache, lens, scale)
        lk, lv = pkg.kv4_load(cache, ints([0] * B, device), cap)
        check_attention(out, q.float()[:, :, None], lk.float().cpu(), lv.float().cpu(), lens.tolist(), scale, what=f"kv4 {step}")
        if int(lens[0]) == cap:
            held = [t.clone() for t in (K, V, *cache)]
            index, new = pkg.kv_select(weights, lens, keep, sinks=4, recent=8, weights_out=weights, lens=lens)
            assert new.tolist() == [keep] * B
            pkg.kv_compact((K, V), index, lens)
            pkg.kv_compact(cache, index, lens)
            at = index.long()[..., None]
            for t, old in zip((K, V, *cache), held):
                assert torch.equal(t[:, :, :keep], old.gather(2, at.expand(-1, -1, -1, t.size(3))))
            assert (weights[:, :, keep:] == 0).all() and (weights[:, :, :keep] > 0).all()
    # every step spread one unit of weight per q head over the positions, and evictions took some away
    assert (weights.sum((1, 2)) <= 50 * NKV * G + 1e-2).all()


@pytest.mark.parametrize("kind,T,lens,splits", [
    ("window", 1, [4000, 1, 0, 37, 3999], 0), ("window", 1, [1] * 7 + [6000], 3), ("window", 5, [4000, 2500, 3, 0, 900, 17], 2),
    ("tracked", 1, [4000, 1200, 0, 64, 2000, 5], 0), ("tracked", 1, [6000] * 4, 7), ("kv4", 3, [9000, 4, 0, 5000, 31], 2),
    ("kv4", 1, [16000, 15999, 1, 8000], 4), ("window", 9, [3000, 17, 0, 2900], 2),
])
def test_splits_dealt_by_length(device, kind, T, lens, splits):
    """A batch of long rows of very different lengths (also none at all): the splits of a launch go to the rows by length. Every
    row against the oracle, and what it gets alone."""
    rng = np.random.default_rng(len(lens) + T)
    B, NKV, G, D, cap = len(lens), 1, 4, 128, max(lens) + 5
    q = randn(rng, B, NKV * G, T, D)
    k, v = randn(rng, B, NKV, cap, D), randn(rng, B, NKV, cap, D)
    starts = [min(7 * b, n) for b, n in enumerate(lens)]
    qd, kd, vd, ld, sd = q.to(device), k.to(device), v.to(device), ints(lens, device), ints(starts, device)
    qd, kw = qd if T > 1 else qd[:, :, 0], dict(kv_start=sd, num_splits=splits)
    if kind == "window":
        out = pkg.gqa_window(qd, kd, vd, ld, D ** -0.5, 0, **kw)
    elif kind == "kv4":
        cache = pkg.kv4_store(kd, vd, pkg.kv4_cache(B, NKV, cap, D, device), ints([0] * B, device))
        k, v = (x.cpu() for x in pkg.kv4_load(cache, ints([0] * B, device), cap))
        out = pkg.gqa_decode_kv4(qd, cache, ld, D ** -0.5, **kw)
    else:
        w, wo = torch.rand(B, NKV, cap, device=device), torch.full((B, NKV, cap), -3.0, device=device)
        out = pkg.gqa_decode_tracked(qd, kd, vd, ld, D ** -0.5, w, weights_out=wo, **kw)
        for b, n in enumerate(lens):
            grown = wo[b, 0, starts[b]:n].double() - w[b, 0, starts[b]:n].double()
            # fp32 sums of a weight below 5 (2^-22 each) and of probabilities (their errors below 2^-16 relative)
            assert abs(float(grown.sum()) - (G if n > starts[b] else 0)) <= n * 2.0 ** -22 + G * 2.0 ** -16, b
            assert (wo[b, 0, :starts[b]] == -3).all() and (wo[b, 0, n:] == -3).all(), b
    check_attention(out, q.float(), k.float(), v.float(), lens, D ** -0.5, starts=starts, what=f"{kind} {lens}")


def test_tracked_splits_share_a_workspace(device):
    """One split writes no partials; a call of several that follows in the same workspace still finds its counters zero."""
    rng = np.random.default_rng(12)
    B, NKV, G, D, cap = 2, 2, 2, 64, 700
    q, k, v = (randn(rng, *s).to(device) for s in ((B, NKV * G, D), (B, NKV, cap, D), (B, NKV, cap, D)))
    lens, w = ints([700, 300], device), torch.zeros(B, NKV, cap, device=device)
    ws = pkg.long_workspace("tracked", device, B, NKV * G, NKV, D, cap, num_splits=5)
    for splits in (5, 1, 5, 1, 3):
        wo = torch.full_like(w, 7.0)
        out = pkg.gqa_decode_tracked(q, k, v, lens, D ** -0.5, w, weights_out=wo, num_splits=splits, workspace=ws)
        check_attention(out, q.float().cpu()[:, :, None], k.float().cpu(), v.float().cpu(), [700, 300], D ** -0.5,
                        what=f"{splits} splits")
        assert abs(float(wo[1, :, :300].sum()) - NKV * G) < 1e-3 and (wo[1, :, 300:] == 7).all(), splits


def test_calls_of_all_sizes_share_the_streams_workspace(device):
    """Batches, heads, chunk lengths and splits in turn on one stream, which keeps one workspace a kind for them."""
    from breeze_tts_2_flash_amd import long_cache
    rng = np.random.default_rng(21)
    cases = [(1, 1, 2, 64, 1, 900, 0), (3, 2, 4, 128, 2, 700, 5), (1, 8, 2, 128, 200, 1200, 3), (1, 2, 1, 64, 40, 800, 2),
             (2, 1, 8, 128, 5, 600, 7), (1, 8, 8, 64, 600, 1500, 2), (4, 2, 2, 64, 1, 2000, 0)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for again in range(2):
            for B, NKV, G, D, T, n, splits in cases + cases[::-1]:
                q, k, v = randn(rng, B, NKV * G, T, D), randn(rng, B, NKV, n, D), randn(rng, B, NKV, n, D)
                lens = [n - 100 * b for b in range(B)]
                out = pkg.gqa_window(q.to(device), k.to(device), v.to(device), ints(lens, device), D ** -0.5, 0, num_splits=splits)
                check_attention(out, q.float(), k.float(), v.float(), lens, D ** -0.5, what=f"{again} {B} {NKV} {G} {D} {T}")
    side.synchronize()
    assert len([key for key in long_cache._WS if key[1] == side.cuda_stream]) <= 2  # few units, and chunks of more


def _calls(device, seed):
    """One call of each kind on inputs of its own: (name, run(workspaces), state to vary)."""
    rng = np.random.default_rng(seed)
    B, NKV, G, D, cap = 2, 2, 2, 128, 1500
    q, k, v = (x.to(device) for x in (randn(rng, B, NKV * G, D), randn(rng, B, NKV, cap, D), randn(rng, B, NKV, cap, D)))
    lens = ints([1500, 900], device)
    cache = pkg.kv4_store(k, v, pkg.kv4_cache(B, NKV, cap, D, device), ints([0, 0], device))
    weights = torch.from_numpy(rng.random((B, NKV, cap)).astype(np.float32)).to(device)
    wo, outs, ws = torch.zeros_like(weights), [torch.zeros_like(k), torch.zeros_like(v)], {}
    for kind in ("window", "kv4", "tracked"):
        ws[kind] = pkg.long_workspace(kind, device, B, NKV * G, NKV, D, cap, window=700 if kind == "window" else 0, sinks=4)

    def run(use_ws):
        w = lambda kind: ws[kind] if use_ws else None  # noqa: E731
        a = pkg.gqa_window(q, k, v, lens, D ** -0.5, 700, sinks=4, workspace=w("window"))
        b = pkg.gqa_decode_kv4(q, cache, lens, D ** -0.5, workspace=w("kv4"))
        c = pkg.gqa_decode_tracked(q, k, v, lens, D ** -0.5, weights, weights_out=wo, workspace=w("tracked"))
        index, n = pkg.kv_evict((k, v), wo, lens, 600, sinks=4, recent=50, outs=outs, weights_out=torch.zeros_like(wo))
        lk, lv = pkg.kv4_load(cache, lens - 900, 17)
        return [a, b, c, wo, index, n, *outs, lk, lv]
    return run, q, lens


def test_captured_and_replayed(device):
    run, q, lens = _calls(device, 4)
    run(True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run(True)
    gen = torch.Generator().manual_seed(7)
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=gen).to(BF16))
        lens.copy_(ints([1500 - 31 * i, 901 + i], device))
        g.replay()
        torch.cuda.synchronize()
        held = [t.clone() for t in got]
        want = run(False)
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b), i


def test_capture_without_workspace_raises(device):
    rng = np.random.default_rng(4)
    q, k = randn(rng, 1, 2, 128).to(device), randn(rng, 1, 2, 5000, 128).to(device)
    lens = ints([5000], device)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="workspace"):
        with torch.cuda.graph(g, stream=side):
            pkg.gqa_window(q, k, k, lens, 0.1, 0)
    torch.cuda.synchronize()


def test_capture_takes_no_stream_workspace(device):
    """Two graphs captured on a stream that has a workspace of its own: each needs one passed, so that both may run at once."""
    rng = np.random.default_rng(6)
    k = randn(rng, 1, 2, 5000, 128).to(device)
    lens, side = ints([5000], device), torch.cuda.Stream()
    qs = [randn(rng, 1, 4, 128).to(device) for _ in range(2)]
    outs, graphs = [torch.empty_like(q) for q in qs], [torch.cuda.CUDAGraph() for _ in qs]
    ws = [pkg.long_workspace("window", device, 1, 4, 2, 128, 5000) for _ in qs]
    want = [pkg.gqa_window(q, k, k, lens, 0.1, 0) for q in qs]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        pkg.gqa_window(qs[0], k, k, lens, 0.1, 0)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="workspace"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            pkg.gqa_window(qs[0], k, k, lens, 0.1, 0)
    torch.cuda.synchronize()
    for q, o, g, w in zip(qs, outs, graphs, ws):
        with torch.cuda.graph(g, stream=side):
            for _ in range(8):
                pkg.gqa_window(q, k, k, lens, 0.1, 0, o, workspace=w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, x) for o, x in zip(outs, want))


def test_two_streams(device):
    """Calls in flight on two streams do not share workspaces."""
    a, b = _calls(device, 1), _calls(device, 2)
    want = [[t.clone() for t in run(False)] for run, _, _ in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(6):
        for j, (s, (run, _, _)) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[j].append([t.clone() for t in run(False)])
    torch.cuda.synchronize()
    for j in range(2):
        for r in got[j]:
            assert all(torch.equal(x, y) for x, y in zip(r, want[j]))


def test_compiled(device):
    run, q, lens = _calls(device, 3)
    rng = np.random.default_rng(0)
    k, v = randn(rng, 2, 2, 1500, 128).to(device), randn(rng, 2, 2, 1500, 128).to(device)
    weights = torch.rand(2, 2, 1500, device=device)

    def step(q, k, v, lens, weights):
        cache = pkg.kv4_store(k, v, pkg.Kv4Cache(*(torch.zeros(2, 2, 1500, n, dtype=torch.uint8, device=q.device)
                                                   for n in (64, 64, 4, 4))), lens * 0)
        a = pkg.gqa_window(q, k, v, lens, 0.1, 100, sinks=2) + pkg.gqa_decode_kv4(q, cache, lens, 0.1)
        w = torch.zeros_like(weights)
        b = pkg.gqa_decode_tracked(q, k, v, lens, 0.1, weights, weights_out=w)
        index, n = pkg.kv_select(w, lens, 300, recent=10)
        ko, vo = pkg.kv_compact((k, v), index, n, (torch.zeros_like(k), torch.zeros_like(v)))
        return a, b, w, index, n, ko, vo

    want = step(q, k, v, lens, weights)
    got = torch.compile(step, fullgraph=True)(q, k, v, lens, weights)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_refusals(device):
    rng = np.random.default_rng(0)
    q, k = randn(rng, 2, 4, 128).to(device), randn(rng, 2, 2, 64, 128).to(device)
    lens, w = ints([5, 6], device), torch.zeros(2, 2, 64, device=device)
    cache = pkg.kv4_cache(2, 2, 64, 128, device)
    bad = [
        lambda: pkg.gqa_window(q, k, k, lens, 0.1, -1), lambda: pkg.gqa_window(q, k, k, lens, 0.1, 2**31),
        lambda: pkg.gqa_window(q, k, k, lens, 0.1, 8, sinks=-1), lambda: pkg.gqa_window(q.float(), k, k, lens, 0.1, 8),
        lambda: pkg.gqa_window(q, k, k[:, :, :32], lens, 0.1, 8), lambda: pkg.gqa_window(q, k[..., :64], k[..., :64], lens, 0.1, 8),
        lambda: pkg.gqa_window(q, k, k, lens.long(), 0.1, 8), lambda: pkg.gqa_window(q, k, k, lens, 0.1, 8, kv_start=lens[:1]),
        lambda: pkg.gqa_window(q, k, k, lens, 0.1, 8, torch.empty(2, 4, 64, dtype=BF16, device=device)),
        lambda: pkg.gqa_window(q, k, k, lens, 0.1, 8, num_splits=300),
        lambda: pkg.gqa_window(q, k, k, lens, 0.1, 8, num_splits=4, workspace=torch.zeros(16, dtype=torch.uint8, device=device)),
        lambda: pkg.gqa_decode_kv4(q[..., :64].contiguous(), cache, lens, 0.1),
        lambda: pkg.gqa_decode_kv4(randn(rng, 2, 4, 17, 128).to(device), cache, lens, 0.1),
        lambda: pkg.gqa_decode_kv4(q, cache._replace(k_scale=cache.k_scale[:, :, :32]), lens, 0.1),
        lambda: pkg.kv4_store(k, k, cache, lens[:1]), lambda: pkg.kv4_store(k[:, :1], k[:, :1], cache, lens),
        lambda: pkg.kv4_store(k, k[:, :, ::2], cache, lens), lambda: pkg.kv4_load(cache, lens, 3, k, k),
        lambda: pkg.gqa_decode_tracked(q, k, k, lens, 0.1, w[:, :, :32]),
        lambda: pkg.gqa_decode_tracked(q, k, k, lens, 0.1, w.double()),
        lambda: pkg.gqa_decode_tracked(randn(rng, 2, 4, 2, 128).to(device), k, k, lens, 0.1, w),
        lambda: pkg.gqa_decode_tracked(q, k, k, lens, 0.1, w, weights_out=w[:, :1].expand(2, 2, 64)),
        lambda: pkg.kv_select(w, lens, 65), lambda: pkg.kv_select(w, lens, 0), lambda: pkg.kv_select(w, lens, 8, sinks=5, recent=4),
        lambda: pkg.kv_compact((k, k.clone(), k.clone(), k.clone(), k.clone()), ints([[[0]] * 2] * 2, device), lens),
        lambda: pkg.kv_compact((k,), ints([[[0]] * 2] * 2, device), lens, (k.float(),)),
    ]
    codes = lambda n: torch.zeros(2, 1, 64, n, dtype=torch.uint8, device=device).expand(2, 2, 64, n)  # noqa: E731
    both = torch.empty(3, dtype=torch.int32, device=device)
    bad += [
        lambda: pkg.gqa_window(q, k, k, lens, 0.1, 8, torch.empty(2, 1, 128, dtype=BF16, device=device).expand(2, 4, 128)),
        lambda: pkg.kv4_store(k, k, pkg.Kv4Cache(codes(64), codes(64), cache.k_scale, cache.v_scale), lens),
        lambda: pkg.kv4_store(k, k, cache._replace(k_scale=codes(4), v_scale=codes(4)), lens),
        lambda: pkg.kv4_store(k, k, cache._replace(v=cache.k), lens),
        lambda: pkg.kv4_load(cache, lens, 64, k, k),
        lambda: pkg.kv4_load(cache, lens, 4, *(k[:, :1, :4].expand(2, 2, 4, 128), k[:, 1:, :4].expand(2, 2, 4, 128))),
        lambda: pkg.kv_select(w, both[:2], 8, lens=both[1:]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
