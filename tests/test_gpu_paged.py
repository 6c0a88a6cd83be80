"""GPU: rotary positions and the paged cache (include/bz_paged_cache.h) against their float64 oracles. Tolerances are
oracle.long_cache.attention_bound's and oracle.paged.turn_bound's (derived there); codes, scales and copied values are compared
exactly."""
import numpy as np
import pytest
import torch

import breeze_tts_2_flash_amd as pkg
from oracle.paged import attention_bound, f8_round, norm, paged_attention, place_of, tokens_of, turn, turn_bound

pytestmark = pytest.mark.gpu

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


def ints(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def randn(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(BF16)


def f64(t):
    return t.double().cpu().numpy()


# ------------------------------------------------------------------------------------------------------ rope

ROPE_CASES = [
    # tokens, heads, head_dim, rotary, interleaved, scaling, first position
    (1, 1, 128, 128, False, None, 0), (2, 40, 128, 128, False, None, 1000), (3, 5, 64, 64, True, "linear", 5),
    (17, 3, 128, 16, False, "ntk", 100000), (33, 7, 64, 48, True, "yarn", 1048576), (5, 9, 128, 112, False, "yarn", 131072),
    (64, 1, 64, 16, True, None, 4000000), (257, 6, 128, 64, True, "linear", 262143),
]


@pytest.mark.parametrize("case", ROPE_CASES, ids=str)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_rope_against_oracle(device, case, dtype):
    N, H, D, R, inter, scaling, first = case
    rng = np.random.default_rng(N + H)
    x = randn(rng, N, H, D)
    pos = torch.from_numpy(first + rng.integers(0, 7, N)).to(dtype)
    f = pkg.rope_frequencies(R, 10000.0, device, interleaved=inter, scaling=scaling, factor=4.0 if scaling else 1.0, trained=8192)
    out = pkg.rope(x.to(device), pos.to(device), f)
    back = pkg.rope(x.to(device), pos.to(device), f, inverse=True)
    torch.cuda.synchronize()
    freq = f64(f.inv_freq)
    want, undo = turn(f64(x), pos, freq, f.factor, inter), turn(f64(x), pos, freq, f.factor, inter, inverse=True)
    assert (np.abs(f64(out) - want) <= turn_bound(f64(x), want, freq, f.factor, inter)).all()
    assert (np.abs(f64(back) - undo) <= turn_bound(f64(x), undo, freq, 1 / f.factor, inter)).all()
    assert torch.equal(out[..., R:].cpu(), x[..., R:])


def test_rope_layouts(device):
    """q and k as a view of a projection's output, in place, into a wider tensor, and by no tokens or heads."""
    rng = np.random.default_rng(3)
    f = pkg.rope_frequencies(64, 1e6, device)
    qkv = randn(rng, 7, 12, 64).to(device)
    pos = torch.arange(7, device=device)
    held = qkv.clone()
    want = pkg.rope(held[:, :10].contiguous(), pos, f)
    x = qkv[:, :10]
    assert pkg.rope(x, pos, f, x) is x
    assert torch.equal(x, want) and torch.equal(qkv[:, 10:], held[:, 10:])
    wide = torch.full((10, 7, 72), 3.0, dtype=BF16, device=device)
    pkg.rope(held[:, :10], pos, f, wide.transpose(0, 1)[..., :64])
    assert torch.equal(wide.transpose(0, 1)[..., :64], want) and (wide[..., 64:] == 3).all()
    assert pkg.rope(held[:0, :10], pos[:0], f).shape == (0, 10, 64) and pkg.rope(held[:, :0], pos, f).shape == (7, 0, 64)
    one = held[:1, :1].expand(7, 10, 64)  # a broadcast input
    assert torch.equal(pkg.rope(one, pos, f), pkg.rope(one.contiguous(), pos, f))


# ---------------------------------------------------------------------------------------------------- stores

class Batch:
    """Rows with `new` tokens behind `past` positions each, their pages at random, `spare` tokens of no row at the end."""

    def __init__(self, rng, past, new, page_size, NKV, D, device, bits=16, spare=0, extra_pages=2, first=0):
        self.past, self.new = past, new
        self.lens = [p + n for p, n in zip(past, new)]
        self.q_start = [first + sum(new[:b]) for b in range(len(new) + 1)]
        self.N = self.q_start[-1] + spare
        need = [-(-n // page_size) for n in self.lens]
        self.pages = sum(need) + extra_pages
        order, at = rng.permutation(self.pages), 0
        self.table = np.full((len(new), max(max(need), 1) + 1), -1, np.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.page_size, self.NKV, self.D, self.bits, self.device = page_size, NKV, D, bits, device

    def cache(self):
        return pkg.paged_cache(self.pages, self.NKV, self.page_size, self.D, self.device, F8 if self.bits == 8 else BF16)

    def args(self):
        return torch.from_numpy(self.table).to(self.device), ints(self.lens, self.device)

    def starts(self):
        return ints(self.q_start, self.device)


STORE_CASES = [
    # past, new, page, NKV, D
    ([0], [1], 16, 1, 128), ([15, 16, 0], [1, 1, 1], 16, 8, 128), ([0, 5, 40], [33, 0, 7], 32, 2, 64),
    ([100, 3], [70, 129], 64, 3, 128), ([7, 0, 1000], [1, 260, 2], 256, 4, 64),
]


@pytest.mark.parametrize("case", STORE_CASES, ids=str)
@pytest.mark.parametrize("bits", [8, 16])
def test_paged_store_and_load(device, case, bits):
    """Every value where it belongs, and no other place touched."""
    past, new, page, NKV, D = case
    rng = np.random.default_rng(D + page)
    b = Batch(rng, past, new, page, NKV, D, device, bits, spare=3)
    k, v = randn(rng, b.N, NKV, D), randn(rng, b.N, NKV, D)
    k[0, 0] *= 1000
    v[0] *= 1e-30
    if b.N > 6:
        k[1, 0, 5], v[2, 0, 1], k[3] = float("nan"), float("inf"), 0
    cache = b.cache()
    for x in cache:
        if x is not None:
            x.view(torch.uint8).fill_(99)
    held = [None if x is None else x.clone() for x in cache]
    table, lens = b.args()
    assert pkg.paged_store(k.to(device), v.to(device), cache, table, lens, b.starts()) is cache
    out = pkg.paged_load(cache, table, ints([p for p in past], device), max(new))
    torch.cuda.synchronize()
    want = [x.clone() for x in held if x is not None]
    places = {n: place_of(b.table, page, b.pages, *rp) for n, rp in tokens_of(b.lens, b.q_start).items()}
    for i, x in enumerate((k, v)):
        values, codes, E = f8_round(f64(x))
        for n, (pg, at) in places.items():
            if bits == 8:
                want[i].view(torch.uint8)[pg, :, at] = torch.from_numpy(codes[n]).to(device)
                want[2 + i][pg, :, at] = torch.from_numpy(E[n]).to(device)
            else:
                want[i][pg, :, at] = x[n].to(device)
        for row in range(len(new)):
            for t in range(new[row]):
                n = b.q_start[row] + t
                got = f64(out[i][row, :, t])
                np.testing.assert_array_equal(got, values[n] if bits == 8 else f64(x[n]))
            assert (out[i][row, :, -(-b.lens[row] // page) * page - past[row]:] == 0).all()  # no page there
    for got, exp in zip([x for x in cache if x is not None], want):
        assert torch.equal(got.view(torch.uint8), exp.view(torch.uint8))


def test_store_rounding_of_8_bits(device):
    """Ties, the borders of a scale, subnormals, and every magnitude of a bf16 value."""
    rows = [[448, 449, 464, -448, 1.0625, 1.1875, 2 ** -10, 3 * 2 ** -10] * 8, [450] + [2 ** -9] * 63, [0.0, -0.0] * 32, [1e-40] * 64,
            [-1.75] + [1 / 3] * 63, [1.7578125] + [-1 / 3] * 63]
    rows += [[2.0 ** e * (1 + (i % 128) / 128) * (-1) ** i / 2 ** (i % 12) for i in range(64)] for e in range(-120, 120, 7)]
    x = torch.tensor(rows, dtype=torch.float64).to(BF16)[:, None]
    n = len(rows)
    cache = pkg.paged_cache(1, 1, 64, 64, device, F8)
    pkg.paged_store(x.to(device), x.to(device), cache, ints([[0]], device), ints([n], device), ints([0, n], device))
    values, codes, E = f8_round(f64(x))
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        assert np.array_equal(s[0, 0, :n].cpu().numpy(), E[:, 0])
        assert np.array_equal(c.view(torch.uint8)[0, 0, :n].cpu().numpy(), codes[:, 0])
    k, _ = pkg.paged_load(cache, ints([[0]], device), ints([0], device), n)
    np.testing.assert_array_equal(f64(k)[0, 0], values[:, 0])


@pytest.mark.parametrize("case", STORE_CASES, ids=str)
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("normed,inter,rotary", [(True, False, 1.0), (False, True, 0.5), (True, True, 0.25)])
def test_rope_store(device, case, bits, normed, inter, rotary):
    past, new, page, NKV, D = case
    G, R = 2, int(D * rotary)
    rng = np.random.default_rng(D + page + bits)
    b = Batch(rng, past, new, page, NKV, D, device, bits, spare=2, first=1 if len(new) > 1 else 0)
    qkv = randn(rng, b.N, (G + 2) * NKV, D)
    q, k, v = qkv.split([G * NKV, NKV, NKV], 1)
    weights = [(1 + 0.2 * randn(rng, D).float()).to(BF16) if normed else None for _ in range(2)]
    f = pkg.rope_frequencies(R, 1e6, device, interleaved=inter, scaling="yarn", factor=4.0, trained=512)
    cache, (table, lens) = b.cache(), b.args()
    d = qkv.to(device)
    dq, dk, dv = d.split([G * NKV, NKV, NKV], 1)
    out = torch.full((b.N, G * NKV, D), 5.0, dtype=BF16, device=device)
    dw = [None if w is None else w.to(device) for w in weights]
    assert pkg.rope_store(dq, dk, dv, cache, table, lens, f, b.starts(), out, q_norm_weight=dw[0], k_norm_weight=dw[1]) is out
    ck, cv = pkg.paged_load(cache, table, ints(past, device), max(new))
    own = pkg.rope_store(dq, dk, dv, cache, table, lens, f, b.starts(), dq, q_norm_weight=dw[0], k_norm_weight=dw[1])  # in place
    torch.cuda.synchronize()
    where = tokens_of(b.lens, b.q_start)
    mine = sorted(where)
    pos = [where[n][1] for n in mine]
    freq = f64(f.inv_freq)
    wants = []
    for x, w in ((q, weights[0]), (k, weights[1])):
        y = f64(x)[mine] if w is None else norm(f64(x)[mine], f64(w), 1e-6)
        z = turn(y, pos, freq, f.factor, inter)
        # the norm's error: D + 4 roundings of 2^-24 in the sum, the root and two products
        wants.append((z, turn_bound(y, z, freq, f.factor, inter) + (D + 4) * 2.0 ** -24 * (np.abs(y) + np.abs(z))))
    got = f64(out)
    assert (np.abs(got[mine] - wants[0][0]) <= wants[0][1]).all()
    assert (got[[n for n in range(b.N) if n not in where]] == 5).all()
    assert torch.equal(own[mine], out[mine]) and own is dq
    vv = f64(v)
    for i, n in enumerate(mine):
        row, p = where[n]
        z, bound = wants[1][0][i], wants[1][1][i]
        if bits == 8:  # half a step of the code (2^-4 of it, or of a subnormal 2^-10 of the scale, under max / 224) in place of bf16's
            bound = bound + 2.0 ** -4 * np.abs(z) + 2.0 ** -10 / 224 * np.abs(z).max(-1, keepdims=True)
        assert (np.abs(f64(ck[row, :, p - past[row]]) - z) <= bound).all()
        np.testing.assert_array_equal(f64(cv[row, :, p - past[row]]), f8_round(vv[n])[0] if bits == 8 else vv[n])


def test_rope_store_positions(device):
    """Positions of its own, in either type; then the pages hold what rope and paged_store would have put there."""
    rng = np.random.default_rng(8)
    b = Batch(rng, [3, 20], [4, 30], 16, 2, 64, device)
    q, k, v = (randn(rng, b.N, h, 64).to(device) for h in (4, 2, 2))
    f = pkg.rope_frequencies(64, 1e4, device)
    table, lens = b.args()
    for pos in (torch.arange(b.N, device=device) * 1000, torch.arange(b.N, device=device, dtype=torch.int32) - 5):
        one, two = b.cache(), b.cache()
        out = pkg.rope_store(q, k, v, one, table, lens, f, b.starts(), positions=pos)
        pkg.paged_store(pkg.rope(k, pos, f), v, two, table, lens, b.starts())
        assert torch.equal(out, pkg.rope(q, pos, f))
        assert torch.equal(one.k, two.k) and torch.equal(one.v, two.v)


# ------------------------------------------------------------------------------------------------- attention

def filled(b, rng, spread=1.0):
    """A cache whose rows hold random values and whose other places hold NaN, and the values that it stands for."""
    k, v = (randn(rng, b.pages, b.NKV, b.page_size, b.D) for _ in range(2))
    k[:, :, ::13] *= 4
    v *= spread
    used = np.zeros((b.pages, b.page_size), bool)
    for row, n in enumerate(b.lens):
        for p in range(n):
            at = place_of(b.table, b.page_size, b.pages, row, p)
            if at is not None:
                used[at] = True
    out = torch.from_numpy(~used)[:, None]
    if b.bits == 16:
        k, v = (x.masked_fill(out[..., None], float("nan")) for x in (k, v))
        return pkg.PagedCache(k.to(b.device), v.to(b.device)), f64(k), f64(v)
    made, values = [], []
    for x in (k, v):
        val, codes, E = f8_round(f64(x))
        E = np.where(out.numpy(), 255, E)
        values.append(np.where(out.numpy()[..., None], np.nan, val))
        made.append((torch.from_numpy(codes).to(b.device).view(F8), torch.from_numpy(E).to(torch.uint8).to(b.device)))
    return pkg.PagedCache(made[0][0], made[1][0], made[0][1], made[1][1]), *values


def check(out, q, k, v, b, scale, G, chunked=None, what=""):
    ref, spread, reach = paged_attention(f64(q), k, v, b.table, b.lens, b.q_start, scale)
    got = f64(out)
    where = tokens_of(b.lens, b.q_start)
    few = 16 // G
    for n, (row, _) in where.items():
        one_term = b.new[row] > few if chunked is None else chunked
        bound = attention_bound(ref[n], spread[n], reach[n], scale, b.D, one_term)
        assert np.isfinite(got[n]).all(), f"{what}: token {n} of row {row} is not finite"
        excess = np.abs(got[n] - ref[n]) - bound
        assert excess.max() <= 0, f"{what}: token {n} of row {row}: {excess.max():.3e} past the bound"
    return ref


FEW_CASES = [
    # past, new, page, NKV, G, D
    ([0], [1], 16, 1, 1, 128), ([15, 300, 0], [1, 1, 1], 16, 2, 2, 128), ([1023, 700], [1, 1], 16, 8, 2, 128),
    ([60, 1, 500, 77], [1, 1, 1, 1], 32, 1, 8, 64), ([5000, 100, 17], [1, 1, 1], 64, 1, 4, 128), ([100, 33, 0, 2], [3, 0, 5, 1], 16, 2, 2, 64),
    ([2000, 511, 9], [2, 1, 4], 256, 4, 4, 128), ([300] * 70, [1, 2] * 35, 16, 1, 1, 64), ([31, 200] * 3, [8, 8] * 3, 32, 2, 2, 128),
    ([3000], [16], 128, 1, 1, 128), ([900, 40], [2, 2], 1024, 2, 8, 64),
    # 17 to 64 columns: two sets a workgroup
    ([100, 700, 5], [9, 3, 16], 16, 2, 2, 128), ([2000, 31], [8, 5], 64, 1, 8, 64), ([500], [20], 32, 1, 1, 128), ([1], [17], 16, 1, 1, 64),
    ([40, 900, 0], [5, 5, 2], 16, 2, 4, 64), ([1000, 3, 70], [16, 1, 0], 16, 1, 4, 128), ([5000, 64], [33, 64], 256, 2, 1, 64),
    ([300] * 70, [3, 8] * 35, 16, 1, 4, 64),
]


@pytest.mark.parametrize("case", FEW_CASES, ids=lambda c: f"rows{len(c[0])}new{max(c[1])}p{c[2]}kv{c[3]}g{c[4]}d{c[5]}")
@pytest.mark.parametrize("bits", [8, 16])
def test_few_tokens(device, case, bits):
    past, new, page, NKV, G, D = case
    rng = np.random.default_rng(page + D + len(new))
    b = Batch(rng, past, new, page, NKV, D, device, bits, spare=1 if max(new) > 1 else 0)
    cache, k, v = filled(b, rng)
    q = randn(rng, b.N, NKV * G, D)
    out = torch.full((b.N, NKV * G, D), 9.0, dtype=BF16, device=device)
    table, lens = b.args()
    single = max(new) == min(new) == 1
    assert pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, None if single else b.starts(), out,
                         max_tokens=max(new)) is out
    torch.cuda.synchronize()
    check(out, q, k, v, b, D ** -0.5, G, False)
    assert (out[b.q_start[-1]:] == 9).all()


@pytest.mark.parametrize("rows,longest,NKV,G,D,hint", [
    (130, 200, 8, 2, 64, 0), (130, 200, 8, 2, 128, 1), (260, 90, 4, 1, 128, 5000), (70, 40, 32, 1, 64, 40),  # so many that rows stay whole
    (1, 900, 300, 1, 64, 0), (3, 700, 520, 1, 64, 0), (5, 300, 300, 1, 64, 0), (2, 60, 1100, 1, 64, 0)])  # more kv heads than CUs
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("ragged", [False, True])
def test_many_units(device, rows, longest, NKV, G, D, hint, bits, ragged):
    rng = np.random.default_rng(rows + NKV)
    past = [int(x) for x in rng.integers(0, longest, rows)]
    new = [1] * rows
    if ragged:
        new[0] = 2
    b = Batch(rng, past, new, 16, NKV, D, device, bits)
    cache, k, v = filled(b, rng)
    q = randn(rng, b.N, NKV * G, D)
    table, lens = b.args()
    out = pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts() if ragged else None, max_tokens=2, max_seq_len=hint)
    torch.cuda.synchronize()
    check(out, q, k, v, b, D ** -0.5, G, False)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0, float("nan")])
@pytest.mark.parametrize("T,NKV,G,D,past", [(1, 2, 2, 128, 400), (12, 2, 2, 64, 400), (150, 8, 8, 64, 0), (300, 8, 8, 128, 0), (60, 8, 8, 128, 2500)])
@pytest.mark.parametrize("bits", [8, 16])
def test_scales(device, scale, T, NKV, G, D, past, bits):
    """Scales of either sign and zero; one that is NaN makes every output NaN but those of tokens that attend nothing."""
    rng = np.random.default_rng(T)
    b = Batch(rng, [past, 0], [T, T], 32, NKV, D, device, bits)
    b.lens[1] = T // 2
    cache, k, v = filled(b, rng)
    q = randn(rng, b.N, NKV * G, D)
    table, lens = b.args()
    out = pkg.gqa_paged(q.to(device), cache, table, lens, scale, b.starts())
    torch.cuda.synchronize()
    none = b.q_start[1] + T - T // 2  # the tokens up to here of the second row attend nothing
    assert (out[b.q_start[1]:none] == 0).all()
    if scale != scale:
        assert out[:b.q_start[1]].isnan().all() and out[none:].isnan().all()
    else:
        check(out, q, k, v, b, scale, G, True)


CHUNK_CASES = [
    # past, new, page, NKV, G, D
    ([0], [129], 16, 1, 1, 128), ([0, 0], [64, 17], 16, 2, 2, 128), ([500, 3, 0], [100, 33, 260], 32, 2, 4, 64),
    ([1500], [70], 64, 8, 2, 128), ([0, 900, 77, 300], [200, 1, 2, 1], 16, 2, 2, 128), ([4000, 10], [40, 0], 256, 1, 8, 64),
    ([63, 64, 65], [65, 64, 63], 64, 2, 1, 64), ([700, 20, 0, 5, 1], [9, 300, 1, 1, 17], 16, 4, 4, 128), ([0], [1000], 128, 2, 2, 128),
    ([10] * 70, [20, 1] * 35, 16, 1, 2, 64),
    # as many columns as the chunk kernels take: one, two and four column groups a workgroup, and positions split
    ([0, 700], [100, 60], 16, 8, 8, 64), ([1500, 300], [60, 9], 32, 8, 8, 128), ([0, 33, 7], [100, 90, 130], 16, 8, 8, 64),
    ([200, 90], [150, 140], 64, 8, 8, 128), ([9], [400], 16, 8, 4, 128), ([0, 17], [800, 790], 16, 8, 8, 64),
    ([40], [1560], 64, 8, 8, 64), ([3000, 77], [110, 100], 16, 8, 4, 128), ([6000], [70], 256, 8, 8, 64), ([5000, 1, 2500], [40, 0, 50], 16, 16, 4, 128),
    ([2100, 900, 30, 600], [90, 1, 100, 2], 16, 8, 8, 128), ([0, 33, 7], [200, 190, 130], 16, 8, 8, 64), ([0], [1540], 64, 8, 8, 128),
]


@pytest.mark.parametrize("case", CHUNK_CASES, ids=lambda c: f"rows{len(c[0])}new{max(c[1])}p{c[2]}kv{c[3]}g{c[4]}d{c[5]}")
@pytest.mark.parametrize("bits", [8, 16])
def test_chunks(device, case, bits):
    past, new, page, NKV, G, D = case
    rng = np.random.default_rng(page + D + len(new))
    b = Batch(rng, past, new, page, NKV, D, device, bits, spare=2)
    cache, k, v = filled(b, rng)
    q = randn(rng, b.N, NKV * G, D)
    out = torch.full((b.N, NKV * G, D), 9.0, dtype=BF16, device=device)
    table, lens = b.args()
    pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts(), out)
    torch.cuda.synchronize()
    check(out, q, k, v, b, D ** -0.5, G, None if len(new) > 1 else True, "device's choice")
    assert (out[b.q_start[-1]:] == 9).all()
    # the same batch by the kernel for few tokens (the hint steers, and nothing else)
    pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts(), out, max_tokens=1)
    torch.cuda.synchronize()
    check(out, q, k, v, b, D ** -0.5, G, False, "few")


MIXED_CASES = {
    # chunks and rows of few tokens in one launch; past, new
    "whole": ([0, 300, 20], [1040, 1, 3]), "whole, many rows": ([0] + [17 * i for i in range(39)], [600] + [1, 2, 3] * 13),
    "split": ([2500, 300], [900, 1]), "split, beside rows": ([2500, 300, 900], [400, 1, 1]), "four groups": ([0, 100], [2100, 1]),
    "drafts": ([0, 3000, 2000, 3300], [700, 20, 32, 9]), "drafts, short": ([0] + [40] * 20, [900] + [20, 33] * 10),
    "few in front": ([700, 0, 1500, 33], [2, 500, 8, 300]),
}


@pytest.mark.parametrize("case", MIXED_CASES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", [8, 16])
def test_mixed(device, case, D, bits):
    past, new = MIXED_CASES[case]
    rng = np.random.default_rng(len(new) + D)
    b = Batch(rng, past, new, 32, 8, D, device, bits, spare=2)
    cache, k, v = filled(b, rng)
    q = randn(rng, b.N, 16, D)
    out = torch.full((b.N, 16, D), 9.0, dtype=BF16, device=device)
    table, lens = b.args()
    pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts(), out, max_tokens=max(new), max_seq_len=max(b.lens))
    torch.cuda.synchronize()
    check(out, q, k, v, b, D ** -0.5, 2)
    assert (out[b.q_start[-1]:] == 9).all()
    for _ in range(3):  # the order in which workgroups end changes nothing
        again = torch.full_like(out, 9.0)
        pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts(), again, max_tokens=max(new), max_seq_len=max(b.lens))
        assert torch.equal(again.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("seed", range(60))
def test_random_batches(device, seed):
    """Batches of any rows, page sizes, groups and hints, right or wrong."""
    rng = np.random.default_rng(1000 + seed)
    pick = lambda *a: a[rng.integers(len(a))]  # noqa: E731
    D, bits, page, NKV, G = pick(64, 128), pick(8, 16), pick(16, 32, 64, 512), pick(1, 2, 3, 8), pick(1, 2, 4, 8)
    rows = int(rng.integers(1, 7))
    new = [int(pick(0, 1, 1, 2, 5, rng.integers(1, 40), rng.integers(1, 200))) for _ in range(rows)]
    new[0] = max(new[0], 1)
    past = [int(pick(0, rng.integers(0, 100), rng.integers(0, 1500))) for _ in range(rows)]
    b = Batch(rng, past, new, page, NKV, D, device, bits, spare=int(rng.integers(0, 3)), first=int(rng.integers(0, 2)))
    for _ in range(int(pick(0, 0, 2))):  # a hole
        b.table[rng.integers(rows), rng.integers(b.table.shape[1])] = -1
    cache, k, v = filled(b, rng, spread=float(pick(1.0, 100.0)))
    q = randn(rng, b.N, NKV * G, D)
    out = torch.full((b.N, NKV * G, D), 9.0, dtype=BF16, device=device)
    table, lens = b.args()
    pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts(), out, max_tokens=int(pick(0, 0, max(new), 1, 10)),
                  max_seq_len=int(pick(0, max(b.lens), 50, 100000)))
    torch.cuda.synchronize()
    check(out, q, k, v, b, D ** -0.5, G, True, str((past, new, page, NKV, G, D, bits)))
    assert (out[:b.q_start[0]] == 9).all() and (out[b.q_start[-1]:] == 9).all()


@pytest.mark.parametrize("T,NKV,G,D,past", [(1, 2, 2, 128, 0), (40, 2, 2, 128, 0), (40, 8, 8, 64, 0), (70, 8, 8, 64, 0), (60, 8, 8, 128, 2500),
                                          (80, 8, 8, 128, 0)])
@pytest.mark.parametrize("bits", [8, 16])
def test_holes_and_bad_pages(device, T, NKV, G, D, past, bits):
    """Pages outside the cache in the middle of a row hold nothing; shared pages are read for each; a row of holes gives zeros."""
    rng = np.random.default_rng(T)
    b = Batch(rng, [600 + past, 300, 200, 90], [T] * 4, 16, NKV, D, device, bits)
    b.table[0, 3:9], b.table[0, 20] = -1, b.pages
    b.table[1, :10] = b.table[0, 9:19]  # shared with row 0
    b.table[2, :] = 2 ** 31 - 1
    b.table[3, 2] = b.table[3, 1]  # twice in one row
    b.table[3, 3] = -2 ** 31
    cache, k, v = filled(b, rng)
    q = randn(rng, b.N, NKV * G, D)
    table, lens = b.args()
    out = pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts())
    torch.cuda.synchronize()
    check(out, q, k, v, b, D ** -0.5, G, T > 8)
    assert (out[2 * T:3 * T] == 0).all()


@pytest.mark.parametrize("bits", [8, 16])
def test_rows_without_positions(device, bits):
    """Lengths of zero, below zero, shorter than the chunk, and past the table."""
    rng = np.random.default_rng(5)
    for new, NKV, G in (([1, 1, 1, 1, 1], 1, 2), ([40, 30, 20, 50, 17], 1, 2), ([140, 130, 120, 150, 117], 8, 8), ([900, 700, 1000, 800, 600], 8, 8)):
        b = Batch(rng, [100] * 5, new, 32, NKV, 64, device, bits)
        b.lens = [0, -7, max(new[2] // 2, 1), b.lens[3], 4000]
        cache, k, v = filled(b, rng)
        q = randn(rng, b.N, NKV * G, 64)
        table, lens = b.args()
        out = pkg.gqa_paged(q.to(device), cache, table, lens, 0.125, b.starts())
        torch.cuda.synchronize()
        ref = check(out, q, k, v, b, 0.125, G, max(new) > 8)
        assert (out[:b.q_start[2]] == 0).all() and (ref[:b.q_start[2]] == 0).all()


@pytest.mark.parametrize("T,NKV,G,hint,past", [
    (1, 2, 2, 0, 130), (5, 2, 2, 0, 130), (60, 2, 2, 0, 130), (33, 2, 4, 0, 130), (5, 2, 2, 5, 130), (10, 2, 2, 10, 130), (13, 2, 4, 13, 130),
    (60, 2, 2, 1, 130), (100, 8, 8, 0, 130), (40, 8, 8, 0, 3000), (300, 8, 8, 0, 40)])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_later_tokens_values_stay_out(device, T, NKV, G, hint, past, bits, value):
    """A non-finite value at a token's own position reaches that token and those behind it, and no other."""
    rng = np.random.default_rng(T + G)
    b = Batch(rng, [past, 70], [T, T], 16, NKV, 128, device, bits)
    cache, k, v = filled(b, rng)
    at = T // 2
    pg, pl = place_of(b.table, 16, b.pages, 0, past + at)
    v[pg, 1, pl] = 0  # for the oracle, whose products with 0 would spread it; no token compared attends it
    if bits == 8:
        cache.v_scale[pg, 1, pl] = 255
    else:
        cache.v[pg, 1, pl, 3:5] = value
    q = randn(rng, b.N, NKV * G, 128)
    table, lens = b.args()
    out = pkg.gqa_paged(q.to(device), cache, table, lens, 128 ** -0.5, b.starts(), max_tokens=hint)
    torch.cuda.synchronize()
    ref, spread, reach = paged_attention(f64(q), k, v, b.table, b.lens, b.q_start, 128 ** -0.5)
    got = f64(out)
    clean = np.ones((b.N, NKV * G), bool)
    clean[at:T, G:2 * G] = False
    excess = np.abs(got - ref) - attention_bound(ref, spread, reach, 128 ** -0.5, 128, T > 16 // G and hint == 0)
    assert np.isfinite(got[clean]).all() and excess[clean].max() <= 0
    hit = got[at:T, G:2 * G]
    if bits == 8 or np.isnan(value):
        assert np.isnan(hit[..., 3:5] if bits == 16 else hit).all()
    else:
        assert (hit[..., 3:5] == np.inf).all()
    if bits == 16:
        assert np.isfinite(np.delete(hit, [3, 4], -1)).all()


@pytest.mark.parametrize("T,NKV,G,past", [(1, 1, 2, 200), (30, 1, 2, 200), (150, 8, 8, 200), (60, 8, 8, 4000)])
def test_scores_without_bounds(device, T, NKV, G, past):
    """Scores of -inf give zeros where there are no others, a NaN scale gives NaN, a scale of 0 the mean, a negative one its own."""
    rng = np.random.default_rng(T)
    b = Batch(rng, [past, 0], [T, 0], 32, NKV, 64, device)
    cache, k, v = filled(b, rng)
    q = randn(rng, b.N, NKV * G, 64)
    q[..., 0] = 1
    table, lens = b.args()
    call = lambda c, s: pkg.gqa_paged(q.to(device), c, table, lens, s, b.starts())  # noqa: E731
    for s in (0.0, -0.2):
        out = call(cache, s)
        torch.cuda.synchronize()
        check(out, q, k, v, b, s, G, T > 8)
    assert torch.isnan(call(cache, float("nan"))).all()
    down = cache._replace(k=cache.k.clone())
    down.k[..., 0] = float("-inf")
    assert (call(down, 0.2) == 0).all()


@pytest.mark.parametrize("T,NKV,G", [(1, 2, 2), (3, 2, 2), (50, 2, 2), (100, 8, 8)])
@pytest.mark.parametrize("bits", [8, 16])
def test_layouts(device, T, NKV, G, bits):
    """K and V side by side in one tensor, heads behind positions, strided q and out, a table and lengths in the middle of others."""
    rng = np.random.default_rng(T + bits)
    D = 64
    b = Batch(rng, [150, 33, 64], [T] * 3, 16, NKV, D, device, bits)
    cache, k, v = filled(b, rng)
    raw = [x.view(torch.uint8) for x in cache[:2]] if bits == 8 else list(cache[:2])
    kv = torch.stack(raw, 2).permute(0, 3, 1, 2, 4).contiguous()  # [pages, page_size, NKV, 2, D]
    parts = [kv[:, :, :, i].permute(0, 2, 1, 3) for i in (0, 1)]
    if bits == 8:
        parts = [x.view(F8) for x in parts] + [torch.stack(cache[2:], 1)[:, i] for i in (0, 1)]
    cache = pkg.PagedCache(*parts)
    q = randn(rng, b.N, NKV * G, D)
    wide = torch.zeros(NKV * G, b.N, D + 8, dtype=BF16, device=device)
    wide[..., :D] = q.transpose(0, 1)
    full = torch.full((NKV * G, b.N, D + 1), 7.0, dtype=BF16, device=device)
    table, lens = b.args()
    table = torch.cat([torch.full_like(table, -5), table, table], 1)[:, table.size(1):2 * table.size(1)]
    lens = torch.cat([lens, lens, lens])[3:6]
    pkg.gqa_paged(wide.transpose(0, 1)[..., :D], cache, table, lens, D ** -0.5, b.starts(), full.transpose(0, 1)[..., :D])
    torch.cuda.synchronize()
    check(full.transpose(0, 1)[..., :D], q, k, v, b, D ** -0.5, G, T > 8)
    assert (full[..., D:] == 7).all()


def test_one_after_the_other(device):
    """A prompt in chunks, then decode steps, as a server runs them: rope_store and gqa_paged on one cache against attention over the
    whole at once."""
    rng = np.random.default_rng(21)
    NKV, G, D, page = 2, 2, 128, 16
    steps = [[37, 1, 0], [20, 1, 60], [1, 1, 1], [1, 0, 1]]
    rows = [sum(s[b] for s in steps) for b in range(3)]
    x = [randn(rng, n, (G + 2) * NKV, D) for n in rows]
    f = pkg.rope_frequencies(D, 1e6, device)
    table = ints(np.random.default_rng(1).permutation(3 * 8).reshape(3, 8).tolist(), device)
    for dtype in (BF16, F8):
        cache = pkg.paged_cache(24, NKV, page, D, device, dtype)
        done, outs = [0, 0, 0], [[], [], []]
        for s in steps:
            tokens = torch.cat([x[b][done[b]:done[b] + s[b]] for b in range(3)]).to(device)
            q, k, v = tokens.split([G * NKV, NKV, NKV], 1)
            done = [d + n for d, n in zip(done, s)]
            starts = [0, s[0], s[0] + s[1], sum(s)]
            lens, q_start = ints(done, device), ints(starts, device)
            q = pkg.rope_store(q, k, v, cache, table, lens, f, q_start)
            out = pkg.gqa_paged(q, cache, table, lens, D ** -0.5, q_start)
            for b in range(3):
                outs[b].append(out[starts[b]:starts[b + 1]])
        torch.cuda.synchronize()
        for b in range(3):
            turned = turn(f64(x[b][:, :(G + 1) * NKV]), range(rows[b]), f64(f.inv_freq))
            q, k, v = turned[:, :G * NKV], turned[:, G * NKV:], f64(x[b][:, (G + 1) * NKV:])
            if dtype == F8:
                k, v = f8_round(k)[0], f8_round(v)[0]
            pages = [np.concatenate([a, np.zeros((128 - rows[b], NKV, D))]).reshape(8, page, NKV, D).transpose(0, 2, 1, 3) for a in (k, v)]
            ref, spread, reach = paged_attention(q, *pages, [list(range(8))], [rows[b]], [0, rows[b]], D ** -0.5)
            # beyond the kernel's bound: q and k were rounded to bf16 on the way (2^-8 each of every product of a score; at most twice 2^-4
            # of a few k values of 8 bits on a border, which the norm below does not show)
            got = f64(torch.cat(outs[b]))
            slack = 2 * D ** -0.5 * reach[..., None] * 2.0 ** -7 * spread
            assert (np.abs(got - ref) <= attention_bound(ref, spread, reach, D ** -0.5, D, True) + slack).all()


def test_long_row_and_far_pages(device):
    """A row of 40000 positions among short ones, and pages past 2^31 bytes of a cache."""
    rng = np.random.default_rng(3)
    NKV, G, D, page = 1, 4, 64, 256
    pages = (2 ** 31 + 2 ** 28) // (NKV * page * D * 2)
    k, v = (torch.zeros(pages, NKV, page, D, dtype=BF16, device=device) for _ in range(2))
    need = -(-40000 // page)
    at = np.sort(np.random.default_rng(4).permutation(pages)[:need])
    at[-1] = pages - 1
    small = [torch.randn(need, NKV, page, D, device=device, dtype=torch.float32).to(BF16) for _ in range(2)]
    for to, x in zip((k, v), small):
        to[torch.from_numpy(at).to(device)] = x
    q = randn(rng, 3, NKV * G, D)
    table = np.full((3, need), -1, np.int32)
    table[0], table[1, :2], table[2, :3] = at, at[-2:], at[[0, -1, 5]]
    lens = [40000, 300, 700]
    out = pkg.gqa_paged(q.to(device), pkg.PagedCache(k, v), torch.from_numpy(table).to(device), ints(lens, device), D ** -0.5)
    lk, lv = pkg.paged_load(pkg.PagedCache(k, v), torch.from_numpy(table).to(device), ints([39000, 200, 600], device), 100)
    torch.cuda.synchronize()
    index = {int(p): i for i, p in enumerate(at)}
    local = np.array([[index.get(int(p), -1) for p in row] for row in table])
    ref, spread, reach = paged_attention(f64(q), f64(small[0]), f64(small[1]), local, lens, [0, 1, 2, 3], D ** -0.5)
    assert (np.abs(f64(out) - ref) <= attention_bound(ref, spread, reach, D ** -0.5, D)).all()
    for row, start in enumerate([39000, 200, 600]):
        for got, x in ((lk, small[0]), (lv, small[1])):
            for t in (0, 55, 99):
                pg, pl = place_of(local, page, need, row, start + t)
                assert torch.equal(got[row, :, t], x[pg, :, pl])


# ------------------------------------------------------------------------------------------- streams and graphs

@pytest.mark.parametrize("T,NKV,G", [(1, 2, 2), (60, 2, 2), (100, 8, 8)])
def test_graph_follows_the_device(device, T, NKV, G):
    """A captured step replayed with lengths, tables and tokens changed on the device, with eager work between, each replay against the
    eager result."""
    rng = np.random.default_rng(T)
    D, page, B = 128, 16, 3
    cache = pkg.paged_cache(64, NKV, page, D, device)
    table = ints(np.arange(60).reshape(3, 20).tolist(), device)
    N = B * T
    tokens = randn(rng, N, (G + 2) * NKV, D).to(device)
    lens, q_start = ints([T] * B, device), ints([0, T, 2 * T, 3 * T], device)
    f = pkg.rope_frequencies(D, 1e6, device)
    ws = pkg.paged_workspace(device, D, G, T)
    out = torch.zeros(N, G * NKV, D, dtype=BF16, device=device)

    def step(c, o, **more):
        q, k, v = tokens.split([G * NKV, NKV, NKV], 1)
        q = pkg.rope_store(q, k, v, c, table, lens, f, q_start)
        return pkg.gqa_paged(q, c, table, lens, D ** -0.5, q_start, o, max_tokens=T, **more)

    step(cache, out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, out, workspace=ws)
    with pytest.raises(RuntimeError, match="workspace="), torch.cuda.graph(torch.cuda.CUDAGraph()):
        step(cache, out)
    torch.cuda.synchronize()
    for turn_ in range(4):
        tokens.copy_(randn(rng, N, (G + 2) * NKV, D))
        lens.copy_(ints([T + 60 * turn_, T + 7 * turn_, max(T - turn_, 0)], device))
        table.copy_(torch.randperm(60, device=device, dtype=torch.int32).view(3, 20))
        other = pkg.PagedCache(cache.k.clone(), cache.v.clone())
        graph.replay()
        want = step(other, None)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(cache.k, other.k) and torch.equal(cache.v, other.v)


def test_two_streams_at_once(device):
    """Each stream has a workspace of its own, calls of all sizes share it."""
    rng = np.random.default_rng(1)
    cases = []
    for past, new, NKV, G, D in (([3000, 50], [1, 1], 2, 4, 128), ([100, 2000], [50, 70], 2, 2, 128), ([5000], [1], 1, 8, 64), ([900] * 9, [3] * 9, 8, 2, 64),
                                  ([3000, 9], [100, 1], 8, 8, 128), ([0], [300], 8, 8, 64)):
        b = Batch(rng, past, new, 16, NKV, D, device)
        cache, _, _ = filled(b, rng)
        q = randn(rng, b.N, NKV * G, D).to(device)
        cases.append((q, cache, *b.args(), D ** -0.5, b.starts()))
    wants = [pkg.gqa_paged(*c) for c in cases]
    torch.cuda.synchronize()
    # a whole turn of torch's pool of 32, so that the streams of later tests, which may look at what a stream has kept, are what they were
    streams = [torch.cuda.Stream() for _ in range(32)][:2]
    outs = []
    for turn_ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                n = (turn_ + i) % len(cases)
                outs.append((n, pkg.gqa_paged(*cases[n])))
    torch.cuda.synchronize()
    for n, out in outs:
        assert torch.equal(out, wants[n])


def test_same_bits_every_time(device):
    rng = np.random.default_rng(2)
    b = Batch(rng, [7000, 4000, 20, 900], [1, 133, 100, 2], 16, 8, 128, device)
    cache, _, _ = filled(b, rng)
    q = randn(rng, b.N, 32, 128).to(device)
    first = pkg.gqa_paged(q, cache, *b.args(), 128 ** -0.5, b.starts())
    for _ in range(5):
        assert torch.equal(pkg.gqa_paged(q, cache, *b.args(), 128 ** -0.5, b.starts()), first)


def test_compiled(device):
    rng = np.random.default_rng(6)
    b = Batch(rng, [40, 9], [2, 30], 16, 2, 64, device, 8)
    tokens = randn(rng, b.N, 8, 64).to(device)
    f = pkg.rope_frequencies(64, 1e4, device)
    table, lens = b.args()

    def step(cache):
        q, k, v = tokens.split([4, 2, 2], 1)
        q = pkg.rope(q, torch.arange(b.N, device=device), f)
        q = pkg.rope_store(q, k, v, cache, table, lens, f, b.starts())
        pkg.paged_store(k, v, cache, table, lens - 1, b.starts())
        out = pkg.gqa_paged(q, cache, table, lens, 0.125, b.starts())
        return out, *pkg.paged_load(cache, table, ints([0, 0], device), 39)

    one, two = b.cache(), b.cache()
    want = step(one)
    got = torch.compile(step, fullgraph=True)(two)
    torch.cuda.synchronize()
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    for a, c in zip(one, two):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))


# --------------------------------------------------------------------------------------------------- refusals

def test_refusals(device):
    rng = np.random.default_rng(7)
    b = Batch(rng, [10, 20], [2, 3], 16, 2, 64, device)
    q, k, v = (randn(rng, 5, h, 64).to(device) for h in (4, 2, 2))
    cache, (table, lens), st = b.cache(), b.args(), b.starts()
    f = pkg.rope_frequencies(64, 1e4, device)
    pos = torch.arange(5, device=device)
    c8 = pkg.paged_cache(b.pages, 2, 16, 64, device, F8)
    o = torch.zeros(5, 4, 64, dtype=BF16, device=device)
    bad = [
        lambda: pkg.rope(q.float(), pos, f), lambda: pkg.rope(q, pos.float(), f), lambda: pkg.rope(q, pos[:4], f),
        lambda: pkg.rope(q, pos, f._replace(inv_freq=f.inv_freq.float())), lambda: pkg.rope(q, pos, f._replace(factor=0.0)),
        lambda: pkg.rope(q, pos, pkg.rope_frequencies(128, 1e4, device)), lambda: pkg.rope(q, pos, f._replace(inv_freq=f.inv_freq[:7])),
        lambda: pkg.rope(q[..., :48], pos, f), lambda: pkg.rope(q, pos, f, o[:4]), lambda: pkg.rope(q, pos, f, o[:1].expand(5, 4, 64)),
        lambda: pkg.rope(q[:4], pos[:4], f, q[1:]), lambda: pkg.rope(q.cpu(), pos, f), lambda: pkg.rope(q.view(-1)[4:4 + 256].view(1, 4, 64), pos[:1], f),
        lambda: pkg.rope(q, pos, f, inverse=pos), lambda: pkg.rope(q, pos, f._replace(interleaved=pos)),
        lambda: pkg.paged_store(k, v, cache, table, lens), lambda: pkg.paged_store(k, v[:4], cache, table, lens, st),
        lambda: pkg.paged_store(k, v, cache, table, lens, st[:2]), lambda: pkg.paged_store(k, v, cache, table, lens[:1], st),
        lambda: pkg.paged_store(k, v, cache, table.long(), lens, st), lambda: pkg.paged_store(k.float(), v, cache, table, lens, st),
        lambda: pkg.paged_store(k, v, cache._replace(v=cache.k), table, lens, st), lambda: pkg.paged_store(k, v, c8._replace(v_scale=None), table, lens, st),
        lambda: pkg.paged_store(k, v, cache._replace(k_scale=c8.k_scale, v_scale=c8.v_scale), table, lens, st),
        lambda: pkg.paged_store(k, v, c8._replace(v_scale=c8.k_scale), table, lens, st), lambda: pkg.paged_store(k, v, cache._replace(v=c8.v), table, lens, st),
        lambda: pkg.paged_store(k, v, pkg.PagedCache(cache.k[:, :, :8], cache.v[:, :, :8]), table, lens, st),
        lambda: pkg.paged_store(k, v, pkg.PagedCache(cache.k[:1].expand(4, 2, 16, 64), cache.v[:1].expand(4, 2, 16, 64)), table, lens, st),
        lambda: pkg.rope_store(q, k, v, cache, table, lens, f, st, o[:4]), lambda: pkg.rope_store(q[:, :0], k, v, cache, table, lens, f, st),
        lambda: pkg.rope_store(q, k, v, cache, table, lens, f, st, positions=pos[:3]), lambda: pkg.rope_store(q, k, v, cache, table, lens, f, st, k),
        lambda: pkg.rope_store(q, k, v, cache, table, lens, f, st, q_norm_weight=k), lambda: pkg.rope_store(q[:, :2], k, v, cache, table, lens, f, st, k),
        lambda: pkg.paged_load(cache, table, lens, -1), lambda: pkg.paged_load(cache, table, lens[:1], 3), lambda: pkg.paged_load(cache, table, lens, 3, k),
        lambda: pkg.paged_load(cache, table, lens, 3, *[torch.zeros(2, 2, 3, 64, dtype=BF16, device=device)] * 2),
        lambda: pkg.gqa_paged(q, cache, table, lens, 0.1), lambda: pkg.gqa_paged(q[:, :3], cache, table, lens, 0.1, st),
        lambda: pkg.gqa_paged(q.repeat(1, 8, 1), cache, table, lens, 0.1, st), lambda: pkg.gqa_paged(q, cache, table, lens, 0.1, st, q),
        lambda: pkg.gqa_paged(q, cache, table, lens, 0.1, st, o[:4]), lambda: pkg.gqa_paged(q, cache, table, lens, 0.1, st, max_tokens=-1),
        lambda: pkg.gqa_paged(q, cache, table, lens, "x", st), lambda: pkg.gqa_paged(q, cache, table[:, 0], lens, 0.1, st),
        lambda: pkg.gqa_paged(q, cache, table, lens, 0.1, st, workspace=torch.zeros(8, dtype=torch.uint8, device=device)),
        lambda: pkg.paged_cache(4, 2, 24, 64, device), lambda: pkg.paged_cache(4, 2, 16, 96, device), lambda: pkg.paged_cache(4, 2, 16, 64, device, torch.float16),
    ]
    before = [x.clone() for x in (q, k, v, cache.k, cache.v, o)]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(before, (q, k, v, cache.k, cache.v, o)))


def test_no_tokens(device):
    """A batch without tokens is a call like any other."""
    b = Batch(np.random.default_rng(0), [10, 20], [0, 0], 16, 2, 64, device)
    cache, (table, lens), st = b.cache(), b.args(), b.starts()
    f = pkg.rope_frequencies(64, 1e4, device)
    q, k = torch.zeros(0, 4, 64, dtype=BF16, device=device), torch.zeros(0, 2, 64, dtype=BF16, device=device)
    assert pkg.rope_store(q, k, k, cache, table, lens, f, st).shape == (0, 4, 64)
    assert pkg.paged_store(k, k, cache, table, lens, st) is cache
    assert pkg.gqa_paged(q, cache, table, lens, 0.1, st).shape == (0, 4, 64)
    assert pkg.paged_load(cache, table, lens, 0)[0].shape == (2, 2, 0, 64)
    # rows without tokens beside padding alone
    out = torch.full((3, 4, 64), 2.0, dtype=BF16, device=device)
    pkg.gqa_paged(torch.ones_like(out), cache, table, lens, 0.1, st, out)
    assert (out == 2).all()
