"""GPU: calls of the paged cache's operators (include/bz_paged_cache.h) that their documentation allows, or that they refuse, beyond
those of test_gpu_paged.py (whose batches, caches and bounds these use)."""
import numpy as np
import pytest
import torch

import breeze_tts_2_flash_amd as pkg
from tests.test_gpu_paged import BF16, Batch, check, filled, ints, randn

pytestmark = pytest.mark.gpu


def wide_table(b, pages):
    """The batch's table with room for `pages` pages a row, none behind those it has."""
    b.table = np.concatenate([b.table, np.full((len(b.new), pages - b.table.shape[1]), -1, np.int32)], 1)
    return b


# ----------------------------------------------------------------------------------- one row in a bucket of tokens

@pytest.mark.parametrize("T,NKV,G,D,past", [(1, 8, 2, 128, 60), (1, 8, 2, 64, 60), (8, 8, 2, 128, 20), (2, 2, 8, 64, 60), (1, 8, 1, 128, 900),
                                            (4, 8, 4, 128, 0)])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("hint", [0, 300])
def test_single_row_of_few_tokens_in_a_bucket(device, T, NKV, G, D, past, bits, hint):
    """A row of up to 16 / G tokens meets V as two terms also where it is the only one and the rest is padding."""
    rng = np.random.default_rng(T + D + past)
    b = wide_table(Batch(rng, [past], [T], 16, NKV, D, device, bits, spare=300 - T), 256)
    cache, k, v = filled(b, rng)
    q = randn(rng, b.N, NKV * G, D)
    out = torch.full((b.N, NKV * G, D), 9.0, dtype=BF16, device=device)
    table, lens = b.args()
    pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts(), out, max_tokens=hint)
    torch.cuda.synchronize()
    check(out, q, k, v, b, D ** -0.5, G, False)
    assert (out[T:] == 9).all()


@pytest.mark.parametrize("bits", [8, 16])
def test_bucket_of_one_row_captured(device, bits):
    """One captured step of 300 tokens' room, replayed with one token, a few, and all of them."""
    rng = np.random.default_rng(bits)
    NKV, G, D, N = 8, 2, 128, 300
    b = wide_table(Batch(rng, [500], [N], 16, NKV, D, device, bits), 128)
    cache, k, v = filled(b, rng)
    q = randn(rng, N, NKV * G, D)
    dq, out, ws = q.to(device), torch.zeros(N, NKV * G, D, dtype=BF16, device=device), pkg.paged_workspace(device, D, G)
    table, lens = b.args()
    starts = b.starts()
    call = lambda o, **more: pkg.gqa_paged(dq, cache, table, lens, D ** -0.5, starts, o, **more)  # noqa: E731
    call(out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, workspace=ws)
    for n, T in ((61, 1), (800, 300), (33, 8), (0, 1), (700, 30), (700, 0), (64, 1)):
        b.lens, b.new, b.q_start = [n], [T], [0, T]
        lens.copy_(ints([n], device))
        starts.copy_(ints([0, T], device))
        out.fill_(9)
        want = torch.full_like(out, 9.0)
        graph.replay()
        call(want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        check(out, q, k, v, b, D ** -0.5, G)
        assert (out[T:] == 9).all()


# --------------------------------------------------------------------------------------- chunks beside many rows

@pytest.mark.parametrize("past,new,NKV,G,D", [([8000] + [300] * 20, [1700] + [1] * 20, 8, 2, 128),
                                              ([300] * 17 + [5000], [2] * 17 + [800], 4, 4, 128), ([9000] + [300] * 40, [1700] + [1] * 40, 8, 2, 64)])
@pytest.mark.parametrize("bits", [8, 16])
def test_a_chunk_is_split_beside_many_rows(device, past, new, NKV, G, D, bits):
    """A chunk behind a long past is split over positions however many rows of few tokens the batch has: its splits' sums are in the
    workspace (behind those of the rows of few tokens, which take a ninth of it)."""
    rng = np.random.default_rng(len(past))
    b = Batch(rng, past, new, 32, NKV, D, device, bits)
    cache, k, v = filled(b, rng)
    q = randn(rng, b.N, NKV * G, D)
    table, lens = b.args()
    ws = pkg.paged_workspace(device, D, G)
    out = pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts(), max_tokens=max(new), max_seq_len=max(b.lens), workspace=ws)
    torch.cuda.synchronize()
    assert ws[ws.numel() // 2:].any()
    check(out, q, k, v, b, D ** -0.5, G)


# -------------------------------------------------------------------------------------------- holes in the table

@pytest.mark.parametrize("past,new,page,NKV,G,D,hole", [
    ([700], [300], 16, 8, 8, 128, 5), ([700, 40], [300, 90], 32, 8, 8, 64, 7), ([0], [150], 16, 8, 8, 64, 3), ([300], [110], 64, 8, 8, 128, 2),
    ([3000], [110], 16, 8, 8, 128, 100), ([40], [300], 16, 8, 2, 128, 21)])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("which", [-1, 1 << 20])
def test_a_hole_is_not_read_from_another_page(device, past, new, page, NKV, G, D, hole, bits, which):
    """What other pages hold (page 0 above all, and what an earlier call left behind on the chip) changes not a bit where the table has a
    hole, neither -1 nor a number past the cache."""
    rng = np.random.default_rng(D + hole)
    b = Batch(rng, past, new, page, NKV, D, device, bits)
    b.table = np.where(b.table >= 0, b.table + 1, -1).astype(np.int32)  # page 0 is nobody's
    b.pages += 1
    b.table[0, hole] = which
    cache, k, v = filled(b, rng)  # NaN wherever no row lies: in page 0, and where the hole's page would be
    q = randn(rng, b.N, NKV * G, D)
    table, lens = b.args()
    call = lambda c: pkg.gqa_paged(q.to(device), c, table, lens, D ** -0.5, b.starts())  # noqa: E731
    call(pkg.PagedCache(*(None if x is None else x.clone().view(torch.uint8).fill_(255).view(x.dtype) for x in cache)))  # all NaN
    out = call(cache)
    torch.cuda.synchronize()
    check(out, q, k, v, b, D ** -0.5, G, True)
    clean = [x.clone() if x is not None else None for x in cache]
    for x, z in zip(clean, (0, 0, 127, 127)):
        if x is not None:
            x.view(torch.uint8)[0] = z
    assert torch.equal(call(pkg.PagedCache(*clean)), out)


# --------------------------------------------------------------------------------------------------------- flags

def test_flags_are_bools(device):
    """inverse and interleaved: True, False, 1 or 0. Texts, lists and tensors are refused, eager or compiled, not taken for their truth."""
    rng = np.random.default_rng(5)
    b = Batch(rng, [10], [5], 16, 2, 64, device)
    q, k, v = (randn(rng, 5, h, 64).to(device) for h in (4, 2, 2))
    cache, (table, lens), st = b.cache(), b.args(), b.starts()
    f = pkg.rope_frequencies(64, 1e4, device)
    pos = torch.arange(5, device=device)
    held = cache.k.clone()
    for flag in ("no", "false", "", [], [0], None, 2, -1, 1.0, pos[1:2], pos[:1], 1 << 80):
        for call in (lambda: pkg.rope(q, pos, f, inverse=flag), lambda: pkg.rope(q, pos, f._replace(interleaved=flag)),
                     lambda: pkg.rope_store(q, k, v, cache, table, lens, f._replace(interleaved=flag), st)):
            with pytest.raises(RuntimeError, match="must be a bool"):
                call()
    torch.cuda.synchronize()
    assert torch.equal(cache.k, held)
    for flag in (False, True):
        assert torch.equal(pkg.rope(q, pos, f, inverse=flag), pkg.rope(q, pos, f, inverse=int(flag)))
        assert torch.equal(pkg.rope(q, pos, f._replace(interleaved=flag)), pkg.rope(q, pos, f._replace(interleaved=int(flag))))
    assert not torch.equal(pkg.rope(q, pos, f, inverse=True), pkg.rope(q, pos, f))
    compiled = torch.compile(lambda x, flag: pkg.rope(x, pos, f, inverse=flag))
    assert torch.equal(compiled(q, True), pkg.rope(q, pos, f, inverse=True))
    with pytest.raises(Exception, match="must be a bool"):
        compiled(q, "no")


# ---------------------------------------------------------------------------------------------------- many rows

@pytest.mark.parametrize("rows,heads,D", [(65535, 1, 64), (65536, 1, 64), (70001, 2, 128), (2, 65537, 64)])
@pytest.mark.parametrize("bits", [8, 16])
def test_load_of_many_rows_and_heads(device, rows, heads, D, bits):
    """As many rows as the stores and the attention take, each at a place of its own; rows without a page are zeros."""
    pages = 3 if heads > 2 else 1000
    gen = torch.Generator(device=device).manual_seed(rows)
    cache = pkg.paged_cache(pages, heads, 16, D, device, torch.float8_e4m3fn if bits == 8 else BF16)
    values = []
    for i in range(2):
        x = torch.randint(-15, 16, cache.k.shape, generator=gen, device=device).to(BF16)  # every value one of e4m3's
        cache[i].copy_(x)
        values.append(x)
    table = torch.randint(-1, pages, (rows, 2), generator=gen, device=device, dtype=torch.int32)
    starts = torch.randint(0, 30, (rows,), generator=gen, device=device, dtype=torch.int32)
    k, v = pkg.paged_load(cache, table, starts, 3)
    assert k.shape == (rows, heads, 3, D)
    for t in range(3):
        pos = (starts + t).long()
        page = torch.where(pos < 32, table.gather(1, (pos // 16).clamp(max=1)[:, None])[:, 0], -1)
        for out, x in ((k, values[0]), (v, values[1])):
            want = x[page.clamp(min=0).long(), :, pos % 16].masked_fill(page[:, None, None] < 0, 0)
            assert torch.equal(out[:, :, t], want)


# ------------------------------------------------------------------------------------ each row by its own bound

@pytest.mark.parametrize("seed", range(80))
def test_random_batches_by_each_rows_bound(device, seed):
    """Batches of any rows, page sizes, groups, holes and hints: rows of up to 16 / G tokens by the bound of two terms whatever the hint, all
    of them where the hint gives the batch to the kernel for few tokens, and only the others by that of one."""
    rng = np.random.default_rng(5000 + seed)
    pick = lambda *a: a[rng.integers(len(a))]  # noqa: E731
    D, bits, page, NKV, G = pick(64, 128), pick(8, 16), pick(16, 32, 64, 512), pick(1, 2, 3, 8), pick(1, 2, 4, 8)
    rows = int(pick(1, 1, 2, 3, 6, 30))
    new = [int(pick(0, 1, 1, 2, 5, rng.integers(1, 40), rng.integers(1, 200) if rows < 9 else 3)) for _ in range(rows)]
    new[0] = max(new[0], 1)
    past = [int(pick(0, rng.integers(0, 100), rng.integers(0, 1500))) for _ in range(rows)]
    b = Batch(rng, past, new, page, NKV, D, device, bits, spare=int(pick(0, 2, 300)), first=int(rng.integers(0, 2)))
    if rng.integers(2):
        wide_table(b, b.table.shape[1] + 4096 // page)
    for _ in range(int(pick(0, 0, 2))):  # a hole
        b.table[rng.integers(rows), rng.integers(b.table.shape[1])] = -1
    cache, k, v = filled(b, rng, spread=float(pick(1.0, 100.0)))
    q = randn(rng, b.N, NKV * G, D)
    out = torch.full((b.N, NKV * G, D), 9.0, dtype=BF16, device=device)
    table, lens = b.args()
    hint = int(pick(0, 0, max(new), 1, 10))
    pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts(), out, max_tokens=hint,
                  max_seq_len=int(pick(0, max(b.lens), 50, 100000)))
    torch.cuda.synchronize()
    few = 0 < min(hint or b.N, b.N) * G <= 64
    check(out, q, k, v, b, D ** -0.5, G, False if few else None, str((past, new, page, NKV, G, D, bits, hint)))
    assert (out[:b.q_start[0]] == 9).all() and (out[b.q_start[-1]:] == 9).all()


# ------------------------------------------------------------------------------------------ many heads, many rows

@pytest.mark.parametrize("past,new,spare,NKV,G,D,bits", [
    ([50], [100], 0, 300, 1, 128, 8), ([50], [3], 97, 300, 1, 128, 8), ([700], [1], 99, 520, 1, 64, 16), ([9], [90], 30, 1100, 1, 64, 16),
    ([5000], [100], 0, 200, 1, 64, 16), ([5000, 300], [100, 1], 0, 200, 1, 64, 16), ([5000], [2], 90, 200, 1, 64, 16),
    ([4500], [30], 100, 130, 2, 128, 16)])
def test_chunks_of_many_heads(device, past, new, spare, NKV, G, D, bits):
    """Fewer splits a head than rows or column tiles, or none."""
    rng = np.random.default_rng(NKV)
    b = Batch(rng, past, new, 64, NKV, D, device, bits, spare=spare)
    cache, k, v = filled(b, rng)
    q = randn(rng, b.N, NKV * G, D)
    out = torch.full((b.N, NKV * G, D), 9.0, dtype=BF16, device=device)
    table, lens = b.args()
    pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts(), out)
    torch.cuda.synchronize()
    check(out, q, k, v, b, D ** -0.5, G)
    assert (out[b.q_start[-1]:] == 9).all()


@pytest.mark.parametrize("rows,chunk,NKV,G,D", [(1100, 300, 2, 2, 64), (700, 0, 8, 1, 64), (300, 500, 8, 4, 128), (2500, 0, 1, 4, 64)])
@pytest.mark.parametrize("bits", [8, 16])
def test_ragged_batches_of_many_rows(device, rows, chunk, NKV, G, D, bits):
    """Rows without tokens, of one, and of a few, in any order, beside a chunk or not."""
    rng = np.random.default_rng(rows)
    new = [int(x) for x in rng.integers(0, 4, rows)]
    if chunk:
        new[rows // 3] = chunk
    past = [int(x) for x in rng.integers(0, 90, rows)]
    past[rows // 2] = 2000
    b = Batch(rng, past, new, 16, NKV, D, device, bits, spare=5)
    cache, k, v = filled(b, rng)
    q = randn(rng, b.N, NKV * G, D)
    out = torch.full((b.N, NKV * G, D), 9.0, dtype=BF16, device=device)
    table, lens = b.args()
    pkg.gqa_paged(q.to(device), cache, table, lens, D ** -0.5, b.starts(), out)
    torch.cuda.synchronize()
    check(out, q, k, v, b, D ** -0.5, G)
    assert (out[b.q_start[-1]:] == 9).all()
