"""How exact the attention over the 4-bit cache is: 16-bit rows are rounded once, and
long walks over values of one sign lose no more than the sums that the kernels keep in a
row before they are rounded to nearest."""
import numpy as np
import pytest

import lunelette_b200 as L
from tests import kv4_reference as ref
from tests.test_gpu_kv4 import TYPES, Cache, half_step, tensor, torch  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

# What an output may lose to the tensor cores, which cut their sums towards zero: as much as 64 sums of equal
# terms lose that are cut by 2^-23 of what is summed so far (the last sees all of it, the first 1 / 64), and
# of 16-bit rows as much as 128, 1/64 of an FP16 rounding.
SUMS = {"f32": 64, "bf16": 128, "f16": 128}


def cut(name):
    return (SUMS[name] + 1) / 2 * 2.0 ** -23


def fp32_bound(name, spread, weight, total):
    # A score is off by 2^-21 of sum |q k| (q's parts 2^-22 of the row's largest, FP32 sums), which moves a
    # weight by 2 of that; exponentials and FP32 sums another 2^-20, doubled for the parts' own roundings
    # and merges; the weights' FP16 parts end at 2^-30 of the largest weight.
    e = 2 * spread[..., None] * 2.0 ** -20 + 2.0 ** -18 + cut(name)
    return weight * e + 2.0 ** -30 * total + 1e-30


def check_rounded_once(torch, name, got, want, spread, weight, total):
    """got = round(x) of an x within fp32_bound of want: no rounding to 16 bits but the last."""
    half, e = half_step(torch, name), fp32_bound(name, spread, weight, total)
    bound = half * np.abs(want) + (1 + half) * e
    if name == "f16":
        bound = bound + 2.0 ** -25  # below 2^-14 FP16 values lie 2^-24 apart: half of that
    worst = float((np.abs(got - want) / bound).max())
    assert worst <= 1.0, worst


ROUNDED = [  # type, dim, kv heads, group, counts, lengths: clusters, the list, blocks, a mix of them
    ("f16", 128, 2, 4, [1], [500]),
    ("bf16", 128, 2, 4, [1, 1], [300, 17]),
    ("f16", 64, 1, 8, [1], [90]),
    ("bf16", 64, 3, 16, [1, 2], [130, 45]),
    ("f16", 128, 8, 4, [1] * 40, [400 + 13 * i for i in range(40)]),
    ("bf16", 128, 4, 8, [1] * 60, [100 + 17 * i for i in range(60)]),
    ("f16", 64, 2, 5, [1, 2, 3] * 20, [333 + 7 * i for i in range(60)]),
    ("f16", 128, 1, 4, [200], [1000]),
    ("bf16", 128, 2, 8, [40], [500]),
    ("bf16", 64, 1, 2, [130], [131]),
    ("f16", 64, 2, 5, [130, 1, 0, 17, 3, 1], [131, 500, 64, 640, 2, 1])]


@pytest.mark.parametrize("name,dim,heads,group,counts,lengths", ROUNDED)
def test_16_bit_rows_are_rounded_once(torch, name, dim, heads, group, counts, lengths):  # noqa: F811
    c = Cache(torch, counts, lengths, heads, dim, seed=50 + len(counts))
    held = c.fill(np.random.default_rng(51 + dim))
    query = heads * group
    q = tensor(torch, name, np.random.default_rng(52).standard_normal((c.rows, query * dim)) * 1.5)
    out = torch.zeros_like(q)
    c.attend(name, q, query, dim ** -0.5, out)
    got = out.double().cpu().numpy().reshape(c.rows, query, dim)
    q64 = q.double().cpu().numpy().reshape(c.rows, query, dim)
    for s, (n, length) in enumerate(zip(counts, lengths)):
        r = slice(int(c.offsets[s]), int(c.offsets[s]) + n)
        if n:
            check_rounded_once(torch, name, got[r], *ref.attention(q64[r], *held[s], dim ** -0.5, length - n))
    assert c.status.item() == 0


def walk(torch, name, dim, heads, group, counts, pages, mean, seed, rise=None):  # noqa: F811
    """Sequences of `pages` whole pages each, drawn from eight that hold values around `mean`; with `rise`, each
    of the eight has larger keys than those before, q a mean, and they come in that order. Returns outputs,
    their definition in 64 bits and sum p |v|, [rows, heads, group, dim]."""
    rng = np.random.default_rng(seed)
    held, few = [], 8
    c = Cache(torch, [0], [64 * few], heads, dim, seed=seed, spare=0, layers=1, layer=0)
    for kind in (0, 1):
        x = rng.standard_normal((64 * few, heads, dim)) * (1.0 if kind == 0 else 0.25) + (0.0 if kind == 0 else mean)
        if rise and kind == 0:
            x = x + rise * np.arange(few).repeat(64)[:, None, None]
        codes, d = ref.quantise(x)
        for p in range(64 * few):
            ref.store(c.host[0], dim, p // 64, p % 64, codes[p], d[p], kind)
        held.append(torch.from_numpy(ref.dequantise(codes, d).reshape(few, 64, heads, dim)).cuda())
    c.pool.copy_(torch.from_numpy(c.host.reshape(-1)))
    c.counts, c.lengths, c.stride = list(counts), [64 * pages] * len(counts), pages
    c.table = rng.integers(0, few, (len(counts), pages)).astype(np.int32)
    if rise:
        c.table.sort(1)
    c.offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    c.rows, c.max_count, c.max_length = int(c.offsets[-1]), max(counts), 64 * pages
    c.d_offsets, c.d_table = torch.from_numpy(c.offsets).cuda(), torch.from_numpy(c.table).cuda()
    c.d_lengths = torch.tensor(c.lengths, dtype=torch.int32, device="cuda")
    query, scale = heads * group, dim ** -0.5
    q = tensor(torch, name, rng.standard_normal((c.rows, query * dim)) + (0.5 if rise else 0.0))
    out = torch.zeros_like(q)
    c.attend(name, q, query, scale, out)
    assert c.status.item() == 0
    k, v = held
    want, size = (torch.zeros((c.rows, heads, group, dim), dtype=torch.float64, device="cuda") for _ in range(2))
    for s, n in enumerate(counts):
        rows = q[c.offsets[s]:c.offsets[s] + n].double().reshape(n, heads, group, dim)
        times = torch.from_numpy(np.bincount(c.table[s, :-1], minlength=few).astype(np.float64)).cuda()
        last = int(c.table[s, -1])
        scores = scale * torch.einsum("nhgd,pkhd->nhgpk", rows, k)
        w = torch.exp(scores - scores.amax((-2, -1), keepdim=True))
        seen = torch.arange(64, device="cuda")[None] <= 64 - n + torch.arange(n, device="cuda")[:, None]
        w = torch.cat([w * times[:, None], w[..., last:last + 1, :] * seen[:, None, None, None]], -2)
        w = w / w.sum((-2, -1), keepdim=True)
        values = torch.cat([v, v[last:last + 1]])
        at = slice(int(c.offsets[s]), int(c.offsets[s]) + n)
        want[at] = torch.einsum("nhgpk,pkhd->nhgd", w, values)
        size[at] = torch.einsum("nhgpk,pkhd->nhgd", w, values.abs())
    return out.double().reshape(want.shape), want, size


WALKS = [  # type, dim, kv heads, group, counts, pages of a sequence
    ("f32", 128, 8, 4, [1] * 300, 68),       # 300 sessions of 4352 keys: 69 pages a warp
    ("f32", 128, 8, 4, [1] * 64, 2048),      # 443 pages a warp
    ("f32", 64, 2, 4, [2] * 5, 2048),        # two tiles of rows a warp
    ("f32", 64, 256, 1, [1] * 40, 40),       # shares of several whole items
    ("bf16", 128, 8, 8, [1] * 64, 2048),
    ("f16", 128, 8, 4, [1] * 64, 2048),
    ("f16", 64, 16, 16, [1] * 30, 1500),
    ("f32", 128, 4, 4, [32] * 37, 500),      # blocks of rows, 148 of them
    ("f16", 128, 4, 4, [32] * 37, 2048),
    ("bf16", 64, 4, 4, [32] * 37, 300)]


@pytest.mark.parametrize("name,dim,heads,group,counts,pages", WALKS)
@pytest.mark.parametrize("mean", [2.0, 0.0])
def test_long_walks_keep_their_accuracy(torch, name, dim, heads, group, counts, pages, mean):  # noqa: F811
    got, want, size = walk(torch, name, dim, heads, group, counts, pages, mean, seed=pages + heads)
    # scores here are sums of 128 products of size one, 2^-21 of which moves a weight by under 2^-18; it moves
    # an output only as far as its values differ, 1/8 of their mean here and all of them around zero
    e = cut(name) + 2.0 ** -20 + 2.0 ** -18 * (0.125 if mean else 1.0)
    error = (got - want).abs()
    if name == "f32":
        assert (error.norm() / size.norm()).item() <= e
    else:
        half = half_step(torch, name)
        bound = half * want.abs() + (1 + half) * size * e + (2.0 ** -25 if name == "f16" else 0.0)
        assert (error / bound).max().item() <= 1.0


@pytest.mark.parametrize("name,dim,heads,group,counts,pages", [
    ("f32", 128, 8, 4, [1] * 64, 68), ("f32", 64, 2, 4, [2] * 5, 2048), ("f16", 128, 8, 3, [1] * 64, 136),
    ("bf16", 128, 8, 8, [1] * 64, 136), ("f16", 64, 16, 16, [1] * 30, 300), ("f32", 128, 4, 4, [32] * 37, 50),
    ("f16", 64, 4, 4, [32] * 37, 50)])
@pytest.mark.parametrize("rise", [0.1, 1.0])
def test_long_walks_while_the_maximum_rises(torch, name, dim, heads, group, counts, pages, rise):  # noqa: F811
    """What was taken out of the sums is scaled down with them: eight kinds of pages one after the other, each
    with larger scores than the last."""
    got, want, size = walk(torch, name, dim, heads, group, counts, pages, 2.0, seed=pages, rise=rise)
    # sum |q k| is 128 products of 0.9 and 0.8 + 7 rise on average, times 128^-1/2, and under half as much
    # again in every row: 2^-21 of it, twice, is what moves a weight at most
    e = cut(name) + 2.0 ** -20 + 1.5 * (8.2 + 71 * rise) * 2.0 ** -20
    half = half_step(torch, name) if name != "f32" else 0.0
    bound = half * want.abs() + (1 + half) * size * e + (2.0 ** -25 if name == "f16" else 0.0)
    assert ((got - want).abs() / bound).max().item() <= 1.0


@pytest.mark.parametrize("name,dim,heads,group,counts,lengths,at", [
    ("f32", 64, 16, 4, [1] * 30, [2200] * 30, 100), ("f16", 64, 32, 4, [1] * 30, [2600] * 30, 100),
    ("bf16", 64, 32, 8, [1] * 30, [2600] * 30, 100), ("f16", 128, 2, 8, [1], [300], 100), ("bf16", 128, 1, 2, [2], [70], 69),
    ("f16", 64, 1, 4, [60], [900], 870), ("bf16", 128, 1, 4, [90], [1300], 64)])
def test_a_nan_stays_where_it_is_seen(torch, name, dim, heads, group, counts, lengths, at):  # noqa: F811
    """A NaN in one group of one position's values, pages before the sums are taken out again, and in rows of
    every kernel: those dims of the rows that see it, and nothing else."""
    c = Cache(torch, counts, lengths, heads, dim, seed=70, layers=1, layer=0)
    rng = np.random.default_rng(71)
    k, v = (ref.quantise(rng.standard_normal((64, heads, dim))) for _ in range(2))
    for p in range(64):
        for kind, (codes, d) in ((0, k), (1, v)):
            ref.store(c.host[0], dim, 0, p, codes[p], d[p], kind)
    c.host[0, 1:] = c.host[0, :1]
    for s in range(0, len(counts), 3):
        codes, d = (x[at % 64].copy() for x in v)
        d[0, 1] = np.nan
        ref.store(c.host[0], dim, c.table[s, at // 64], at % 64, codes, d, 1)
    c.pool.copy_(torch.from_numpy(c.host.reshape(-1)))
    query = heads * group
    q = tensor(torch, name, rng.standard_normal((c.rows, query * dim)))
    out = torch.zeros_like(q)
    c.attend(name, q, query, dim ** -0.5, out)
    got = out.double().cpu().numpy().reshape(c.rows, heads, group, dim)
    bad = np.zeros(got.shape, bool)
    for row, s, position in c.rows_of():
        bad[row, 0, :, 32:64] = s % 3 == 0 and position >= at
    assert np.array_equal(np.isnan(got), bad)
    assert c.status.item() == 0


def test_append_and_read_report_every_broken_sequence(torch):  # noqa: F811
    """Sequences that no row's search lands on: one whose offsets descend among others within their bounds,
    and an empty one with a length past the bound, the last of many."""
    for offsets, lengths, bit in (([0, 3, 2, 5], [3, 9, 3], 1), ([0, 2, 2, 4], [2, 129, 2], 1), ([0, 2, 2, 4], [2, 128, 2], 0),
                                  ([0] * 4001 + [2], [1] * 4000 + [2], 0), ([0] * 4001 + [2], [1] * 3999 + [-1, 2], 1)):
        n = len(lengths)
        c = Cache(torch, [1] * n, [1] * n, 1, 64, max_count=3, max_length=128, stride=2)
        c.rows = 5 if n == 3 else 2
        c.d_offsets.copy_(torch.tensor(offsets, dtype=torch.int32))
        c.d_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        x = torch.ones((c.rows, 64), device="cuda")
        c.append("f32", x, x)
        assert c.status.item() == bit, (offsets[:5], "append")
        c.status.zero_()
        c.read("f32", x, None)
        assert c.status.item() == bit, (offsets[:5], "read")


@pytest.mark.parametrize("name,dim,heads,group,rows,skew", [("f32", 128, 8, 4, 2500, 0), ("bf16", 64, 3, 7, 3000, 1),
                                                            ("f16", 128, 1, 40, 1300, 0)])
def test_append_rotates_many_rows_in_place(torch, name, dim, heads, group, rows, skew):  # noqa: F811
    """Blocks that take several rows, with the next values already loaded when a row is written over."""
    c = Cache(torch, [rows - 900, 0, 900], [rows, 0, 1000], heads, dim, layers=1, layer=0)
    query = heads * group
    rng = np.random.default_rng(80)
    qkv = tensor(torch, name, rng.standard_normal((rows, (query + 2 * heads) * dim + skew)))[:, skew:]
    q, k, v = qkv.split([query * dim, heads * dim, heads * dim], 1)
    angle = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(0, dim, 2) / dim)
    tables = [torch.from_numpy(np.concatenate([f(angle)] * 2, 1).astype(np.float32)).cuda() for f in (np.cos, np.sin)]
    out = torch.zeros((rows, query * dim), dtype=q.dtype, device="cuda")
    c.append(name, k, v, q, out, query, tables)
    pool, before = c.pool.clone(), k.clone()
    c.pool.zero_()
    c.append(name, k, v, q, q, query, tables)
    assert torch.equal(q, out) and torch.equal(k, before) and c.status.item() == 0
    held = torch.zeros((rows, heads * dim), dtype=q.dtype, device="cuda")
    again = torch.zeros_like(held)
    c.read(name, held, None)
    c.pool.copy_(pool)
    c.read(name, again, None)
    assert torch.equal(held, again)


def test_a_refused_attention_call_launches_nothing(torch):  # noqa: F811
    """More padded rows than the join of the splits has blocks for; the first sequence's only row would be
    written by the kernel for few rows."""
    heads, dim, query = 256, 64, 4096
    c = Cache(torch, [1, 0, 0, 0, 0], [1, 1, 1, 1, 1], heads, dim, stride=1000, layers=1, layer=0)
    c.rows, c.max_count, c.max_length = 1 << 24, 2, 64000
    q = torch.ones((1, query * dim), device="cuda")
    out = torch.full_like(q, 7.0)
    ws = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")
    assert L.library().lunelette_cuda_kv4_attention(
        c.kv4(), 0, c.descriptor(), L.FLOAT32, q.data_ptr(), q.stride(0), query, 0.1, out.data_ptr(), out.stride(0),
        ws.data_ptr(), 1 << 60, c.status.data_ptr(), c.stream()) == -1
    torch.cuda.synchronize()
    assert (out == 7.0).all()


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("heads,counts,lengths", [(8, [1] * 64, [4352] * 64), (8, [256], [4352]),
                                                  (2, [1, 40, 2, 1, 1, 1], [5000] * 6)])
def test_a_workspace_that_is_too_small_is_refused(torch, name, heads, counts, lengths):  # noqa: F811
    group, dim = 4, 128
    c = Cache(torch, counts, lengths, heads, dim, layers=1, layer=0)
    c.pool.zero_()
    query = heads * group
    need = L.library().lunelette_cuda_kv4_attention_workspace(c.kv4(), c.descriptor(), query)
    assert need > 1 << 16
    q = torch.ones((c.rows, query * dim), dtype=getattr(torch, TYPES[name][1]), device="cuda")
    out = torch.full_like(q, 7.0)
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")

    def call(pointer, size):
        return L.library().lunelette_cuda_kv4_attention(
            c.kv4(), 0, c.descriptor(), TYPES[name][0], q.data_ptr(), q.stride(0), query, 0.1, out.data_ptr(),
            out.stride(0), pointer, size, c.status.data_ptr(), c.stream())

    for pointer, size in ((None, need), (ws.data_ptr(), 0), (ws.data_ptr() + 4, need)):
        assert call(pointer, size) == -1, (pointer, size)
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    # the function goes by the largest of the types: the least that this one takes
    refused, taken = 0, need
    while taken - refused > 1:
        size = (taken + refused) // 2
        if call(ws.data_ptr(), size) == 0:
            taken = size
        else:
            refused = size
    torch.cuda.synchronize()
    assert need // 4 <= taken <= need
    out.fill_(7.0)
    ws.fill_(0x5A)
    assert call(ws.data_ptr(), taken - 1) == -1
    torch.cuda.synchronize()
    assert (out == 7.0).all() and (ws == 0x5A).all()
    assert call(ws.data_ptr(), taken) == 0
    torch.cuda.synchronize()
    assert (out == 0.0).all() and (ws[taken:] == 0x5A).all() and c.status.item() == 0
def test_rotated_infinities_of_q_are_the_definitions(torch):  # noqa: F811
    dim, n = 128, 40
    rng = np.random.default_rng(61)
    x = rng.standard_normal((n, 2, dim)).astype(np.float32)
    for row in range(n):
        x[row, row % 2, rng.integers(dim)] = np.inf * (-1) ** row
    x[0, 0, 3], x[0, 0, 67] = np.inf, np.inf
    x[1, 1, 3], x[1, 1, 67] = np.inf, -np.inf
    angle = np.arange(1, n + 1)[:, None] * 10000.0 ** (-np.arange(0, dim, 2) / dim)  # no sine is zero
    cos, sin = (np.concatenate([f(angle)] * 2, 1).astype(np.float32) for f in (np.cos, np.sin))
    tables = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    c = Cache(torch, [n], [n], 1, dim)
    q = torch.from_numpy(x.reshape(n, -1)).cuda()
    out = torch.zeros_like(q)
    k = torch.ones((n, dim), device="cuda")
    c.append("f32", k, k, q, out, 2, tables)
    got = out.cpu().numpy().reshape(x.shape)
    with np.errstate(invalid="ignore"):
        want = np.stack([ref.rotate(x[i], cos[i].astype(np.float64), sin[i].astype(np.float64)) for i in range(n)])
    assert np.isinf(want).any() and np.isnan(want).any()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isinf(got), np.isinf(want)) and (np.sign(got) == np.sign(want))[np.isinf(want)].all()


def test_a_row_with_an_infinity_has_no_distribution(torch):  # noqa: F811
    """Keys of one sign and a minus infinity in q: every score is minus infinity, which is not a mask."""
    for name in TYPES:
        for counts, lengths in (([1], [100]), ([1] * 40, [900] * 40), ([30], [90])):
            c = Cache(torch, counts, lengths, 1, 64, seed=60)
            for s, n in enumerate(lengths):
                for kind in (0, 1):
                    codes, d = ref.quantise(np.full((1, 64), 1.0))
                    for p in range(n):
                        ref.store(c.host[c.layer], 64, c.table[s, p // 64], p % 64, codes, d, kind)
            c.pool.copy_(torch.from_numpy(c.host.reshape(-1)))
            q = torch.ones((c.rows, 2 * 64), dtype=getattr(torch, TYPES[name][1]), device="cuda")
            q[-1, 70] = -np.inf
            out = torch.zeros_like(q)
            c.attend(name, q, 2, 0.1, out)
            assert out[-1, 64:].isnan().all(), (name, counts)
            out[-1, 64:] = 1.0
            assert torch.isfinite(out).all(), (name, counts)
