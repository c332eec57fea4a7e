"""The 4-bit KV cache on the GPU against its definition in 64 bits: appended
pools bit for bit, rows read back, ragged causal attention, bad tables, strides,
streams, captured graphs, pools past 4 GB, and a run of them with the
framework's projections and head."""
import numpy as np
import pytest

import lunelette_b200 as L
from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": (L.FLOAT32, "float32"), "bf16": (L.BFLOAT16, "bfloat16"), "f16": (L.FLOAT16, "float16")}
SENTINEL = 0xAB


@pytest.fixture(scope="module")
def torch():
    import torch
    torch.cuda.init()
    return torch


def half_step(torch, name):
    return float(torch.finfo(getattr(torch, TYPES[name][1])).eps) / 2


class Cache:
    """A pool on the device with sentinel bytes, and the rows of a call over it."""

    def __init__(self, torch, counts, lengths, heads, dim, layers=2, layer=1, spare=2, pad=0, seed=0, pool=None,
                 max_count=None, max_length=None, stride=None):
        rng = np.random.default_rng(seed + 1000)
        need = [max(0, -(-n // 64)) for n in lengths]
        self.torch, self.heads, self.dim, self.layer, self.layers = torch, heads, dim, layer, layers
        self.counts, self.lengths = list(counts), list(lengths)
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.stride = stride or max(need + [1])
        self.table = np.full((len(counts), self.stride), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.spare = order[at:]
        self.offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.rows = int(self.offsets[-1]) + pad
        block = heads * ref.block_bytes(dim)
        if pool is None:
            pool = np.full((layers, self.pages, heads, ref.block_bytes(dim)), SENTINEL, np.uint8)
        self.host = pool
        self.pool = torch.from_numpy(pool.reshape(-1)).cuda()
        assert L.library().lunelette_cuda_kv4_bytes(layers, self.pages, heads, dim) == layers * self.pages * block
        self.d_offsets = torch.from_numpy(self.offsets).cuda()
        self.d_lengths = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")
        self.d_table = torch.from_numpy(self.table).cuda()
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.max_count = max_count if max_count is not None else max(counts + [0])
        self.max_length = max_length if max_length is not None else max(lengths + [0])

    def kv4(self):
        return L.Kv4(self.pool.data_ptr(), self.layers, self.pages, self.heads, self.dim)

    def descriptor(self):
        return L.Rows(self.rows, len(self.counts), self.d_offsets.data_ptr(), self.d_lengths.data_ptr(),
                      self.d_table.data_ptr(), self.stride, self.max_count, self.max_length)

    def stream(self):
        return self.torch.cuda.current_stream().cuda_stream

    def append(self, name, k, v, q=None, q_out=None, query_heads=0, rope=None, rc=0):
        cos, sin = rope if rope else (None, None)
        got = L.library().lunelette_cuda_kv4_append(
            self.kv4(), self.layer, self.descriptor(), TYPES[name][0], k.data_ptr(), k.stride(0), v.data_ptr(),
            v.stride(0), q.data_ptr() if q is not None else None, q.stride(0) if q is not None else 0, query_heads,
            q_out.data_ptr() if q_out is not None else None, q_out.stride(0) if q_out is not None else 0,
            cos.data_ptr() if rope else None, sin.data_ptr() if rope else None, cos.shape[0] if rope else 0,
            self.status.data_ptr(), self.stream())
        assert got == rc

    def read(self, name, k, v, rc=0):
        assert L.library().lunelette_cuda_kv4_read(
            self.kv4(), self.layer, self.descriptor(), TYPES[name][0], k.data_ptr() if k is not None else None,
            k.stride(0) if k is not None else 0, v.data_ptr() if v is not None else None,
            v.stride(0) if v is not None else 0, self.status.data_ptr(), self.stream()) == rc

    def workspace(self, query_heads):
        need = L.library().lunelette_cuda_kv4_attention_workspace(self.kv4(), self.descriptor(), query_heads)
        # whatever it holds may not matter
        return self.torch.full((max(16, need),), 0xFF, dtype=self.torch.uint8, device="cuda")

    def attend(self, name, q, query_heads, scale, out, workspace=None, rc=0):
        ws = workspace if workspace is not None else self.workspace(query_heads)
        assert L.library().lunelette_cuda_kv4_attention(
            self.kv4(), self.layer, self.descriptor(), TYPES[name][0], q.data_ptr(), q.stride(0), query_heads, scale,
            out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(), self.status.data_ptr(), self.stream()) == rc
        self.torch.cuda.synchronize()

    def rows_of(self):
        """(row, sequence, position) of every row of a sequence."""
        for s, (c, n) in enumerate(zip(self.counts, self.lengths)):
            for i in range(c):
                yield int(self.offsets[s]) + i, s, n - c + i

    def fill(self, rng, ramp=0.0):
        """Random keys and values at every position of every sequence, straight into the host's pool:
        per sequence [length, heads, dim] of the stored values. Keys get `ramp` more from page to page."""
        held = []
        for s, n in enumerate(self.lengths):
            stored = []
            for kind in (0, 1):
                x = rng.standard_normal((n, self.heads, self.dim)) * np.exp2(rng.integers(-1, 2, (1, self.heads, 1)))
                if kind == 0:
                    x = x + ramp * (np.arange(n) // 64)[:, None, None]
                codes, d = ref.quantise(x)
                for p in range(n):
                    ref.store(self.host[self.layer], self.dim, self.table[s, p // 64], p % 64, codes[p], d[p], kind)
                stored.append(ref.dequantise(codes, d))
            held.append(stored)
        self.pool.copy_(self.torch.from_numpy(self.host.reshape(-1)))
        return held


def tensor(torch, name, array):
    return torch.from_numpy(np.ascontiguousarray(array)).cuda().to(getattr(torch, TYPES[name][1]))


def rope_tables(torch, positions, dim, seed=0):
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(0, dim, 2) / dim)
    angle = np.concatenate([angle, angle], 1)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    return cos, sin, (torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda())


def expected_pool(cache, k, v, cos=None, sin=None):
    """The pool after appending float64 rows k, v [rows, heads, dim]; and the stored values of each row."""
    pool = cache.host.copy()
    stored = {}
    for row, s, p in cache.rows_of():
        if p < 0:
            continue
        page = cache.table[s, p // 64]
        r = k[row] if cos is None else ref.rotate(k[row], cos[p].astype(np.float64), sin[p].astype(np.float64))
        stored[row] = []
        for kind, x in ((0, r), (1, v[row])):
            codes, d = ref.quantise(x)
            stored[row].append(ref.dequantise(codes, d))
            if 0 <= page < cache.pages:
                ref.store(pool[cache.layer], cache.dim, page, p % 64, codes, d, kind)
    return pool, stored


SHAPES = [  # type, dim, kv heads, group, counts, lengths, unused rows, rotation
    ("f32", 128, 8, 4, [1], [1], 0, True),
    ("f32", 128, 8, 4, [256], [4352], 0, True),
    ("bf16", 128, 2, 3, [3, 0, 70, 1], [66, 5, 70, 16385], 4, True),
    ("f16", 64, 5, 1, [65, 1, 2], [130, 1, 64], 1, True),
    ("f32", 64, 1, 7, [1] * 40, list(range(1, 41)), 0, False),
    ("bf16", 64, 3, 2, [9], [4], 0, True),  # five rows before position 0
]


@pytest.mark.parametrize("name,dim,heads,group,counts,lengths,pad,rope", SHAPES)
def test_append_is_bit_exact_and_reads_back(torch, name, dim, heads, group, counts, lengths, pad, rope):
    rng = np.random.default_rng(dim + len(counts))
    c = Cache(torch, counts, lengths, heads, dim, pad=pad)
    query = heads * group
    qkv = tensor(torch, name, rng.standard_normal((c.rows, (query + 2 * heads) * dim)) * 3)
    q, k, v = qkv.split([query * dim, heads * dim, heads * dim], 1)
    cos, sin, tables = rope_tables(torch, max(lengths), dim)
    q_out = torch.full((c.rows, query * dim), 7.0, dtype=q.dtype, device="cuda")
    c.append(name, k, v, q, q_out, query, tables if rope else None)
    k64, v64, q64 = (x.double().cpu().numpy().reshape(c.rows, -1, dim) for x in (k, v, q))
    want, stored = expected_pool(c, k64, v64, cos if rope else None, sin)
    got = c.pool.cpu().numpy().reshape(want.shape)
    assert np.array_equal(got, want)
    assert c.status.item() == 0
    got_q = q_out.double().cpu().numpy().reshape(c.rows, query, dim)
    touched = np.zeros(c.rows, bool)
    for row, s, p in c.rows_of():
        if p < 0:
            continue
        touched[row] = True
        turned = ref.rotate(q64[row], cos[p].astype(np.float64), sin[p].astype(np.float64)) if rope else q64[row]
        expect = turned * ref.query_scale(p)
        # rounding to FP32 (2^-24), the FP32 query scale (a logarithm of 2 ulp, a product and a sum:
        # under 2^-22) and its product, then the rounding to the row's type
        bound = np.abs(expect) * (2.0 ** -21 + (half_step(torch, name) if name != "f32" else 0)) + 2.0 ** -24
        assert (np.abs(got_q[row] - expect) <= bound).all()
    assert (got_q[~touched] == 7.0).all()
    k_out = torch.full((c.rows, heads * dim), 7.0, dtype=q.dtype, device="cuda")
    v_out = k_out.clone()
    c.read(name, k_out, v_out)
    for kind, x in ((0, k_out), (1, v_out)):
        x = x.double().cpu().numpy().reshape(c.rows, heads, dim)
        assert (x[~touched] == 7.0).all()
        for row in stored:
            e = torch.from_numpy(stored[row][kind]).to(q.dtype).double().numpy()
            assert np.array_equal(x[row], e)


def test_append_special_groups_bit_exact(torch):
    rng = np.random.default_rng(9)
    heads, dim, n = 2, 128, 24
    c = Cache(torch, [n], [n], heads, dim)
    k = rng.standard_normal((n, heads, dim)).astype(np.float32)
    v = rng.standard_normal((n, heads, dim)).astype(np.float32)
    for x in (k, v):
        x[0] = 0.0
        x[1, :, :32] = -0.0
        x[2] *= np.float32(1e-8)                     # below the grid's first step in part
        x[3] *= np.float32(3e-7)                     # on the grid's first steps
        x[4] *= np.float32(1e5)                      # the largest scale
        x[5] *= np.float32(1e36)
        x[6, 0, 5] = np.nan
        x[7, 1, 70] = np.inf
        x[8, 1, 70] = -np.inf
        x[9, :, :] = 2.5                             # all alike
        x[10, 0, 3], x[10, 0, 9] = 9.0, -9.0         # both signs reach the largest magnitude
        x[11, 0, 9], x[11, 0, 3] = 9.0, -9.0
        x[12, 0, :32] = np.arange(32) / 4 - 4.0      # d = 0.5: quarters lie on the borders
        x[13, 0, :32] = np.arange(32) * 0.1875       # d < 0 and borders
        x[14, 0, :16] = np.nextafter(np.float32(np.arange(16) / 2 - 4 + 0.25), np.float32(9))
        x[14, 0, 16:32] = np.nextafter(np.float32(np.arange(16) / 2 - 4 + 0.25), np.float32(-9))
        x[14, 0, 0] = -4.0
        x[15, 0, :32] = np.float32(1e-42)            # FP32 subnormals
        x[16, 0, :32] = np.float32(65280.0) * np.linspace(-1, 1, 32).astype(np.float32)
        # scales next to the border between two of 8 bits
        for j, m in enumerate((1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 1 + 2.0 ** -8 + 2.0 ** -23, 1 + 2.0 ** -8 - 2.0 ** -23)):
            x[17 + j, 0, :32] = 0.25
            x[17 + j, 0, 4] = -m
    dk, dv = torch.from_numpy(k.reshape(n, -1)).cuda(), torch.from_numpy(v.reshape(n, -1)).cuda()
    c.append("f32", dk, dv)
    want, _ = expected_pool(c, k.astype(np.float64), v.astype(np.float64))
    got = c.pool.cpu().numpy().reshape(want.shape)
    assert np.array_equal(got, want)
    out = torch.zeros((n, heads * dim), device="cuda")
    c.read("f32", out, None)
    out = out.cpu().numpy().reshape(n, heads, dim)
    assert np.isnan(out[6, 0, :32]).all() and np.isfinite(out[6, 0, 32:]).all()
    assert np.isnan(out[7, 1, 64:96]).all() and np.isnan(out[8, 1, 64:96]).all()
    assert np.isfinite(out[9:]).all()


def test_append_next_to_code_borders_bit_exact(torch):
    """Values rotated onto the border between two codes within a few 2^-24 of it: a
    quotient formed in FP32 would fall on either side."""
    rng = np.random.default_rng(10)
    heads, dim, n = 4, 64, 200
    c = Cache(torch, [n], [n], heads, dim)
    d = np.exp2(rng.integers(-3, 4, (n, heads, 1, 1))) * rng.integers(128, 256, (n, heads, 1, 1)) / 128.0
    x = (rng.integers(-8, 7, (n, heads, 2, 32)) + 0.5) * d
    x[..., 3] = -8 * d[..., 0]
    x = x.reshape(n, heads, dim).astype(np.float32)
    steps = rng.integers(-2, 3, x.shape)
    for _ in range(2):
        x = np.where(steps > 0, np.nextafter(x, np.float32(np.inf)), np.where(steps < 0, np.nextafter(x, np.float32(-np.inf)), x))
        steps -= np.sign(steps)
    dx = torch.from_numpy(x.reshape(n, -1)).cuda()
    cos, sin, tables = rope_tables(torch, n, dim)
    c.append("f32", dx, dx, rope=tables)
    want, _ = expected_pool(c, x.astype(np.float64), x.astype(np.float64), cos, sin)
    assert np.array_equal(c.pool.cpu().numpy().reshape(want.shape), want)


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_append_and_read_unaligned_rows(torch, name):
    rng = np.random.default_rng(12)
    heads, dim, n = 3, 128, 5
    c = Cache(torch, [2, 3], [2, 70], heads, dim)
    width = heads * dim
    base = tensor(torch, name, rng.standard_normal((n, 2 * width + 5)))
    k, v = base[:, 1:1 + width], base[:, 3 + width:3 + 2 * width]
    cos, sin, tables = rope_tables(torch, 70, dim)
    q_out = torch.full((n, width + 3), 7.0, dtype=base.dtype, device="cuda")
    c.append(name, k, v, k, q_out[:, 2:2 + width], heads, tables)
    k64, v64 = (x.double().cpu().numpy().reshape(n, heads, dim) for x in (k, v))
    want, stored = expected_pool(c, k64, v64, cos, sin)
    assert np.array_equal(c.pool.cpu().numpy().reshape(want.shape), want)
    assert (q_out[:, :2] == 7.0).all() and (q_out[:, 2 + width:] == 7.0).all()
    out = torch.full((n, width + 1), 7.0, dtype=base.dtype, device="cuda")
    c.read(name, out[:, 1:], None)
    assert (out[:, 0] == 7.0).all()
    for row in stored:
        e = torch.from_numpy(stored[row][0]).to(base.dtype)
        assert torch.equal(out[row, 1:].cpu(), e.reshape(-1))


def test_append_rotates_q_in_place(torch):
    rng = np.random.default_rng(13)
    c = Cache(torch, [3], [40], 2, 64)
    qkv = tensor(torch, "f32", rng.standard_normal((3, 8 * 64)))
    cos, sin, tables = rope_tables(torch, 40, 64)
    out = torch.zeros((3, 4 * 64), device="cuda")
    c.append("f32", qkv[:, 256:384], qkv[:, 384:], qkv[:, :256], out, 4, tables)
    c.append("f32", qkv[:, 256:384], qkv[:, 384:], qkv[:, :256], qkv[:, :256], 4, tables)
    assert torch.equal(qkv[:, :256], out)


def test_rows_that_break_their_bounds_are_skipped_and_reported(torch):
    """A page outside the pool, a length past the bound, a count past the bound,
    offsets that descend: the other sequences' rows land, nothing else changes."""
    rng = np.random.default_rng(14)
    heads, dim = 2, 128
    for fault, bit in (("page", 2), ("negative", 2), ("length", 1), ("count", 1), ("offsets", 1)):
        counts, lengths = [2, 3, 2], [70, 40, 9]
        c = Cache(torch, counts, lengths, heads, dim, max_count=3, max_length=128, seed=3)
        x = tensor(torch, "f32", rng.standard_normal((c.rows, heads * dim)))
        skipped = 1
        if fault == "page":
            c.table[1, 0] = c.pages
        if fault == "negative":
            c.table[1, 0] = -5
        if fault == "length":
            c.d_lengths[1] = 129
        if fault == "count":
            c.max_count = 2
        if fault == "offsets":
            c.d_offsets[1] = 6  # sequence 0 takes rows 0..5, sequence 1 a negative count
        c.d_table.copy_(torch.from_numpy(c.table))
        c.append("f32", x, x)
        x64 = x.double().cpu().numpy().reshape(c.rows, heads, dim)
        c.counts[skipped] = 0
        full = list(c.rows_of())
        c.counts = counts
        want = c.host.copy()
        for row, s, p in full:
            if fault == "offsets" and s == 0:
                continue
            for kind in (0, 1):
                codes, d = ref.quantise(x64[row])
                ref.store(want[c.layer], dim, c.table[s, p // 64], p % 64, codes, d, kind)
        got = c.pool.cpu().numpy().reshape(want.shape)
        assert np.array_equal(got, want), fault
        assert c.status.item() == bit, fault
        out = torch.full((c.rows, heads * dim), 7.0, device="cuda")
        c.status.zero_()
        c.read("f32", out, None)
        assert c.status.item() == bit, fault
        bad = [r for r in range(2, 5)]
        assert (out[bad] == 7.0).all(), fault
        att = torch.full((c.rows, heads * dim), 7.0, device="cuda")
        c.status.zero_()
        c.attend("f32", x, heads, 0.1, att)
        assert c.status.item() == bit, fault
        if bit == 1:
            assert (att[bad] == 7.0).all(), fault
        else:
            assert (att[bad] == 0.0).all(), fault  # its only page is skipped
        assert torch.isfinite(att).all()


def attention_check(torch, c, held, name, group, scale, seed, first=None):
    rng = np.random.default_rng(seed)
    query = c.heads * group
    q = tensor(torch, name, rng.standard_normal((c.rows, query * c.dim)) * 1.5)
    out = torch.full((c.rows, query * c.dim), 7.0, dtype=q.dtype, device="cuda")
    c.attend(name, q, query, scale, out)
    got = out.double().cpu().numpy().reshape(c.rows, query, c.dim)
    q64 = q.double().cpu().numpy().reshape(c.rows, query, c.dim)
    for s, (n, length) in enumerate(zip(c.counts, c.lengths)):
        r = slice(int(c.offsets[s]), int(c.offsets[s]) + n)
        want, *size = (np.concatenate(parts, 1) for parts in zip(*(
            ref.attention(q64[r, h * group:(h + 1) * group], held[s][0][:, h:h + 1].astype(np.float64),
                          held[s][1][:, h:h + 1].astype(np.float64), scale, length - n) for h in range(c.heads))))
        check_rows(torch, name, got[r], want, *size)
    assert (got[int(c.offsets[-1]):] == 7.0).all()
    assert c.status.item() == 0
    again = torch.full_like(out, 7.0)
    c.attend(name, q, query, scale, again)
    assert torch.equal(out, again)
    return q, out


def check_rows(torch, name, got, want, spread, weight, total):
    # A score is off by 2^-21 of sum |q k| at most: q in two FP16 parts (2^-22 of the row's largest,
    # products exact) and FP32 sums; the exponentials and the sums of the softmax by another 2^-20 of the
    # terms. An error e in every score moves a weight by at most 2 e of itself. 16-bit rows may round each
    # weight to 11 bits (2^-12), and every output is rounded to its type.
    e = 2 * spread[..., None] * 2.0 ** -20 + 2.0 ** -18
    if name != "f32":
        e = e + 2.0 ** -11
    # The weights' FP16 parts end on FP16's grid of 2^-24, off by half of that, after the weights were taken
    # times 2^14 or 2^5 (decode kernel, the latter in pages whose scales leave 2^-8..2) or 2^7 (block kernel;
    # the reference maximum is a score the row has seen, so the largest weight is 2^7 at least there too):
    # 2^-30 of the largest weight, which the softmax's sum reaches. Outputs that only weights so small make
    # up keep an absolute accuracy of 2^-30 sum |v|, under the 2^-24 of FP32 sums in which larger weights
    # take part.
    floor = 2.0 ** -30 * total
    bound = weight * e + floor + (np.abs(want) * half_step(torch, name) if name != "f32" else 0) + 1e-30
    if name == "f16":
        bound = bound + 2.0 ** -25  # below 2^-14 FP16 values lie 2^-24 apart, whatever their size: half of that
    worst = float((np.abs(got - want) / bound).max()) if got.size else 0.0
    assert worst <= 1.0, worst  # NaN fails too


ATTENTION = [  # type, dim, kv heads, group, counts, lengths, unused rows
    ("f32", 128, 8, 4, [1], [1], 0),
    ("f32", 128, 8, 4, [1], [64], 0),
    ("f32", 128, 8, 4, [1], [65], 0),
    ("f32", 128, 8, 4, [1], [4352], 0),
    ("f32", 128, 2, 1, [1] * 9, [1, 2, 15, 16, 17, 63, 129, 700, 1025], 2),
    ("bf16", 128, 1, 8, [1, 1, 0, 1], [3000, 77, 400, 191], 0),
    ("f16", 64, 3, 16, [1, 2], [300, 45], 0),
    ("f32", 64, 2, 3, [2, 3, 1, 5], [2, 130, 64, 3], 0),     # two rows before position 0
    ("f32", 128, 2, 4, [2, 4], [129, 700], 0),
    ("bf16", 128, 1, 5, [7, 33], [7, 140], 3),
    ("f32", 128, 8, 4, [64], [192], 0),
    ("f32", 128, 1, 4, [200], [1000], 0),
    ("f16", 64, 2, 5, [130, 1, 0, 17, 3], [131, 500, 64, 640, 2], 5),
    ("bf16", 64, 1, 40, [5, 1], [70, 200], 0),
    ("f32", 64, 1, 1, [300], [300], 0),
    ("f32", 128, 1, 2, [100, 1, 40], [60, 0, 41], 0),        # rows before position 0, an empty cache
    ("f16", 64, 1, 130, [1, 2], [70, 65], 0),                # a group beyond a tile's rows
    ("bf16", 64, 256, 1, [1, 0, 1], [20, 0, 66], 1),         # as many KV heads as there may be
    ("f32", 128, 2, 2, [1] * 150, [1 + 37 * i % 200 for i in range(150)], 0),
    ("f16", 64, 2, 1, ([1] * 9 + [0]) * 40, ([5, 64, 0, 131, 17, 65, 1, 30, 128, 9] * 40), 3),  # 400 sequences
    ("f32", 64, 2, 1, [1] * 200, [0] * 200, 0),              # nothing anywhere
    ("f32", 64, 1, 2, [1] * 299 + [30], [1 + i % 90 for i in range(299)] + [50], 0),
]


@pytest.mark.parametrize("name,dim,heads,group,counts,lengths,pad", ATTENTION)
def test_attention_matches_definition(torch, name, dim, heads, group, counts, lengths, pad):
    c = Cache(torch, counts, lengths, heads, dim, pad=pad, seed=len(counts))
    held = c.fill(np.random.default_rng(sum(lengths) + dim))
    attention_check(torch, c, held, name, group, dim ** -0.5, seed=dim + sum(counts))


def over_shared_pages(torch, counts, lengths, heads, dim, pages, seed):
    """A cache whose sequences hold the same few pages again and again; and what they read."""
    c = Cache(torch, [0], [64 * pages], heads, dim, seed=seed, spare=0)
    (k, v), = c.fill(np.random.default_rng(seed))
    by_page = np.argsort(c.table[0, :pages])  # the sequence's page that lies at a place of the pool
    c.counts, c.lengths = list(counts), list(lengths)
    c.stride = -(-max(lengths) // 64)
    c.table = np.random.default_rng(seed + 1).integers(0, pages, (len(counts), c.stride)).astype(np.int32)
    c.offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    c.rows, c.max_count, c.max_length = int(c.offsets[-1]), max(counts), max(lengths)
    c.d_offsets, c.d_table = torch.from_numpy(c.offsets).cuda(), torch.from_numpy(c.table).cuda()
    c.d_lengths = torch.tensor(c.lengths, dtype=torch.int32, device="cuda")
    k, v = (x.reshape(pages, 64, heads, dim).astype(np.float16) for x in (k, v))  # exact
    return c, [[x[by_page[c.table[s, :-(-n // 64)]]].reshape(-1, heads, dim)[:n] for x in (k, v)]
               for s, n in enumerate(lengths)]


@pytest.mark.parametrize("name,dim,heads,group,counts,lengths", [
    ("f32", 64, 16, 5, [1, 1], [160000, 150001]),                        # more than 64 pages a warp
    ("f16", 128, 2, 1, [1] * 3, [200000, 70, 130001]),
    ("f16", 64, 32, 1, [20] * 5, [6000, 5999, 4097, 5000, 4160]),        # more than 64 pages a block
    ("f32", 128, 4, 4, [32] * 10, [5000] * 10)])
def test_attention_over_pages_held_many_times(torch, name, dim, heads, group, counts, lengths):
    c, held = over_shared_pages(torch, counts, lengths, heads, dim, 8, seed=40)
    attention_check(torch, c, held, name, group, dim ** -0.5, seed=41)


def test_attention_ignores_stale_slots_and_other_pages(torch):
    """Bytes of 0xFF everywhere else: NaN scales in the slots behind the last position,
    in other pages and in the other layer."""
    for counts, lengths in (([1, 1], [100, 3]), ([90, 2], [150, 70])):
        c = Cache(torch, counts, lengths, 2, 128, seed=5)
        c.host[:] = 0xFF
        held = c.fill(np.random.default_rng(6))
        attention_check(torch, c, held, "f32", 4, 0.09, seed=7)


def test_attention_scale_zero_and_negative_and_large_scores(torch):
    c = Cache(torch, [1, 40], [500, 300], 2, 64, seed=8)
    held = c.fill(np.random.default_rng(8))
    for scale in (0.0, -0.125, 2.0):
        attention_check(torch, c, held, "f32", 2, scale, seed=9)


@pytest.mark.parametrize("name,dim", [("f32", 128), ("f16", 64)])
def test_attention_scales_of_all_sizes(torch, name, dim):
    """Groups from FP16's smallest scales to the largest, mixed within pages and apart."""
    rng = np.random.default_rng(21)
    for counts, lengths in (([1, 1, 1], [300, 700, 40]), ([20], [150])):
        c = Cache(torch, counts, lengths, 2, dim, seed=21)
        held = []
        for s, n in enumerate(lengths):
            stored = []
            for kind in (0, 1):
                x = rng.standard_normal((n, 2, dim))
                if kind == 1:  # pages of one size, and pages of all
                    size = np.where(np.arange(n) // 64 % 2 == 0, rng.integers(-18, 11, (2, dim // 32, n)),
                                    rng.integers(-18, 11, (2, dim // 32, 1)))
                    x = x * np.exp2(np.repeat(np.moveaxis(size, 2, 0), 32, 2))
                codes, d = ref.quantise(x)
                for p in range(n):
                    ref.store(c.host[c.layer], dim, c.table[s, p // 64], p % 64, codes[p], d[p], kind)
                stored.append(ref.dequantise(codes, d))
            held.append(stored)
        c.pool.copy_(torch.from_numpy(c.host.reshape(-1)))
        attention_check(torch, c, held, name, 2, 0.1, seed=22)


@pytest.mark.parametrize("name,dim,heads,group,counts,lengths", [
    ("f32", 128, 8, 4, [256], [1500]), ("f32", 128, 1, 4, [32], [1000]), ("f16", 64, 2, 5, [100, 3, 40], [900, 700, 1300]),
    ("f16", 128, 4, 8, [64] * 5, [640] * 5)])
def test_attention_scores_that_rise_from_page_to_page(torch, name, dim, heads, group, counts, lengths):
    """Rows whose maximum rises by a lot in every page, among rows whose maximum never does: what
    is summed up so far is scaled down again and again, while later products are under way."""
    c = Cache(torch, counts, lengths, heads, dim, seed=30)
    held = c.fill(np.random.default_rng(31), ramp=8.0)
    attention_check(torch, c, held, name, group, 0.1, seed=32)


def test_attention_q_range(torch):
    """Rows of q far outside FP16's range, zero rows, and a NaN that stays in its row."""
    c = Cache(torch, [1, 1, 1, 20], [200, 200, 64, 90], 1, 128, seed=11)
    held = c.fill(np.random.default_rng(11))
    rng = np.random.default_rng(12)
    q = rng.standard_normal((c.rows, 2, 128)).astype(np.float32)
    q[0] *= np.float32(1e20)
    q[1] *= np.float32(1e-20)
    q[2] = 0
    q[3, 1, 7] = np.nan
    q[9] *= np.float32(1e7)
    d_q = torch.from_numpy(q.reshape(c.rows, -1)).cuda()
    for scale in (1e-20, 1e-7, 0.08):
        out = torch.zeros_like(d_q)
        c.attend("f32", d_q, 2, scale, out)
        got = out.double().cpu().numpy().reshape(c.rows, 2, 128)
        assert np.isnan(got[3, 1]).all() and np.isfinite(got[3, 0]).all()
        for s, (n, length) in enumerate(zip(c.counts, c.lengths)):
            for i in range(n):
                row = int(c.offsets[s]) + i
                if scale == 0.08 and row in (0, 9) or row == 3:
                    continue  # scores of 1e20 keep no digit
                want, *size = ref.attention(q[row:row + 1].astype(np.float64), held[s][0], held[s][1],
                                                     scale, length - n + i)
                check_rows(torch, "f32", got[row:row + 1], want, *size)


def test_attention_keeps_a_nan_from_rows_that_do_not_see_it(torch):
    """A key with a NaN, and values with a NaN in one group, at a position that only
    the later rows of the call see."""
    for counts, lengths, at in (([2], [70], 69), ([40], [90], 60), ([1], [70], 30), ([90], [200], 140)):
        for kind in (0, 1):
            c = Cache(torch, counts, lengths, 1, 128, seed=14)
            held = c.fill(np.random.default_rng(14))
            codes, d = ref.quantise(np.where(np.arange(128) == 70, np.nan, 1.0)[None])
            ref.store(c.host[c.layer], 128, c.table[0, at // 64], at % 64, codes, d, kind)
            c.pool.copy_(torch.from_numpy(c.host.reshape(-1)))
            q = torch.randn((c.rows, 4 * 128), device="cuda")
            out = torch.zeros_like(q)
            c.attend("f32", q, 4, 0.08, out)
            got = out.double().cpu().numpy().reshape(c.rows, 4, 128)
            first = lengths[0] - counts[0]
            for i in range(c.rows):
                if first + i < at:
                    want, *size = ref.attention(q[i:i + 1].double().cpu().numpy().reshape(1, 4, 128), *held[0],
                                                         0.08, first + i)
                    check_rows(torch, "f32", got[i:i + 1], want, *size)
                elif kind == 0:
                    assert np.isnan(got[i]).all()
                else:
                    assert np.isnan(got[i, :, 64:96]).all() and np.isfinite(got[i, :, :64]).all()
                    assert np.isfinite(got[i, :, 96:]).all()


def test_attention_strided_rows(torch):
    rng = np.random.default_rng(15)
    for counts, lengths in (([1, 2], [100, 40]), ([50], [80])):
        c = Cache(torch, counts, lengths, 2, 128, seed=15)
        held = c.fill(rng)
        q = torch.randn((c.rows, 8 * 128 + 9), device="cuda")[:, 3:3 + 8 * 128]
        out = torch.full((c.rows, 8 * 128 + 5), 7.0, device="cuda")
        c.attend("f32", q, 8, 0.08, out[:, 1:1 + 8 * 128])
        dense = torch.zeros((c.rows, 8 * 128), device="cuda")
        c.attend("f32", q.contiguous(), 8, 0.08, dense)
        assert torch.equal(out[:, 1:1 + 8 * 128], dense)
        assert (out[:, 0] == 7.0).all() and (out[:, 1 + 8 * 128:] == 7.0).all()
        q64 = q.double().cpu().numpy().reshape(c.rows, 8, 128)
        r = int(c.offsets[1])
        want, *size = ref.attention(q64[:r], held[0][0], held[0][1], 0.08, lengths[0] - counts[0])
        check_rows(torch, "f32", dense[:r].double().cpu().numpy().reshape(r, 8, 128), want, *size)


def test_attention_bounds_larger_than_the_rows(torch):
    """max_count and max_length are bounds: much larger ones give the same result."""
    counts, lengths = [1, 30, 2], [300, 200, 70]
    c = Cache(torch, counts, lengths, 2, 128, seed=16, stride=64)
    held = c.fill(np.random.default_rng(16))
    q, out = attention_check(torch, c, held, "f32", 4, 0.1, seed=17)
    c.max_count, c.max_length = 500, 4096
    attention_check(torch, c, held, "f32", 4, 0.1, seed=17)


def test_pool_past_4_gb(torch):
    """Pages whose bytes start past 2^32."""
    heads, dim, pages = 8, 128, 66000  # 4.9 GB
    table = np.array([[65990, 3, 65999]], np.int32)
    pool = torch.zeros(pages * heads * ref.block_bytes(dim), dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(18)
    n = 150
    k, v = (rng.standard_normal((n, heads, dim)).astype(np.float32) for _ in range(2))
    d_k, d_v = (torch.from_numpy(x.reshape(n, -1)).cuda() for x in (k, v))
    arrays = [torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([0, n], [n])] + [torch.from_numpy(table).cuda()]
    cache = L.Kv4(pool.data_ptr(), 1, pages, heads, dim)
    r = L.Rows(n, 1, *(a.data_ptr() for a in arrays), 3, n, n)
    lib, stream = L.library(), torch.cuda.current_stream().cuda_stream
    assert lib.lunelette_cuda_kv4_append(cache, 0, r, L.FLOAT32, d_k.data_ptr(), heads * dim, d_v.data_ptr(),
                                         heads * dim, None, 0, 0, None, 0, None, None, 0, None, stream) == 0
    out = torch.zeros_like(d_k)
    assert lib.lunelette_cuda_kv4_read(cache, 0, r, L.FLOAT32, out.data_ptr(), heads * dim, None, 0, None, stream) == 0
    stored = [ref.dequantise(*ref.quantise(x)) for x in (k, v)]
    assert np.array_equal(out.cpu().numpy().reshape(n, heads, dim), stored[0])
    block = ref.block_bytes(dim) * heads
    assert pool[65990 * block:65991 * block].any() and pool[65999 * block:66000 * block].any()
    for count in (1, n):
        arrays[0][1] = count
        r = L.Rows(n, 1, *(a.data_ptr() for a in arrays), 3, count, n)
        ws = torch.empty(max(16, lib.lunelette_cuda_kv4_attention_workspace(cache, r, heads)), dtype=torch.uint8,
                         device="cuda")
        att = torch.zeros_like(d_k)
        assert lib.lunelette_cuda_kv4_attention(cache, 0, r, L.FLOAT32, d_k.data_ptr(), heads * dim, heads, 0.05,
                                                att.data_ptr(), heads * dim, ws.data_ptr(), ws.numel(), None, stream) == 0
        rows = [0] if count == 1 else [0, 63, 64, n - 1]
        got = att.double().cpu().numpy().reshape(n, heads, dim)
        for i in rows:
            want, *size = ref.attention(k[i:i + 1].astype(np.float64), *stored, 0.05, n - count + i)
            check_rows(torch, "f32", got[i:i + 1], want, *size)


def test_side_stream_and_captured_graph_follow_later_lengths(torch):
    """One decode step captured once: append, attention; replayed as the lengths,
    the rows and the tables' contents move on, two sequences, over a page border."""
    heads, dim, group, steps = 2, 128, 4, 6
    c = Cache(torch, [1, 1], [66, 4], heads, dim, seed=20, max_length=256, stride=4)
    c.table[0, :3], c.table[1, :2] = [4, 0, 2], [1, 3]
    c.d_table.copy_(torch.from_numpy(c.table))
    start = [60, 3]
    rng = np.random.default_rng(21)
    query = heads * group
    cos, sin, tables = rope_tables(torch, 256, dim)
    history = [[np.zeros((0, heads, dim))] * 2 for _ in range(2)]
    qkv = torch.zeros((2, (query + 2 * heads) * dim), device="cuda")
    q_out = torch.zeros((2, query * dim), device="cuda")
    out = torch.zeros((2, query * dim), device="cuda")
    ws = c.workspace(query)
    q, k, v = qkv.split([query * dim, heads * dim, heads * dim], 1)

    def step():
        c.append("f32", k, v, q, q_out, query, tables)
        assert L.library().lunelette_cuda_kv4_attention(
            c.kv4(), c.layer, c.descriptor(), L.FLOAT32, q_out.data_ptr(), query * dim, query, 0.09, out.data_ptr(),
            query * dim, ws.data_ptr(), ws.numel(), c.status.data_ptr(), c.stream()) == 0

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = None
    for t in range(start[0] + steps):
        live = [t + 1, max(0, t + 1 - (start[0] - start[1]))]
        host = rng.standard_normal(qkv.shape).astype(np.float32)
        with torch.cuda.stream(side):
            qkv.copy_(torch.from_numpy(host))
            c.d_lengths.copy_(torch.tensor(live, dtype=torch.int32))
            if t < start[0]:
                step()
            else:
                if graph is None:
                    side.synchronize()
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=side):
                        step()
                graph.replay()
        side.synchronize()
        x = host.astype(np.float64).reshape(2, -1, dim)
        for s in range(2):
            p = live[s] - 1
            if p < 0:
                continue
            rk = ref.rotate(x[s, query:query + heads], cos[p].astype(np.float64), sin[p].astype(np.float64))
            for kind, r in ((0, rk), (1, x[s, query + heads:])):
                history[s][kind] = np.concatenate([history[s][kind], ref.dequantise(*ref.quantise(r))[None]])
            if t >= start[0] - 2:
                rq = q_out[s].double().cpu().numpy().reshape(1, query, dim)
                want, *size = ref.attention(rq, history[s][0], history[s][1], 0.09, p)
                check_rows(torch, "f32", out[s].double().cpu().numpy().reshape(1, query, dim), want, *size)
    assert c.status.item() == 0


@pytest.mark.parametrize("heads,two", [(1, [([1], [4000]), ([1, 1], [3000, 2000])]),
                                       (2, [([1], [9000]), ([1] * 30, [300 + 41 * i for i in range(30)])]),
                                       (2, [([150], [2000]), ([40, 1, 3, 70, 1, 1], [900, 700, 64, 1000, 5, 333])])])
def test_two_graphs_with_a_workspace_each_overlap(torch, heads, two):
    """Two captured attention calls on two streams at once, each with its workspace."""
    calls, group = [], 4
    for seed, (counts, lengths) in enumerate(two):
        c = Cache(torch, counts, lengths, heads, 128, seed=seed)
        held = c.fill(np.random.default_rng(seed))
        q, out = attention_check(torch, c, held, "f32", group, 0.09, seed=seed)
        ws, got, stream = c.workspace(group * heads), torch.zeros_like(out), torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            assert L.library().lunelette_cuda_kv4_attention(
                c.kv4(), c.layer, c.descriptor(), L.FLOAT32, q.data_ptr(), q.stride(0), group * heads, 0.09, got.data_ptr(),
                got.stride(0), ws.data_ptr(), ws.numel(), None, c.stream()) == 0
        calls.append((c, q, out, ws, got, stream, graph))
    torch.cuda.synchronize()
    for _ in range(20):
        for *_, got, stream, graph in calls:
            with torch.cuda.stream(stream):
                got.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, _, got, _, _ in calls:
        assert torch.equal(out, got)


def test_refusals_leave_outputs(torch):
    c = Cache(torch, [1, 30], [70, 40], 2, 128)
    c.fill(np.random.default_rng(1))
    q = torch.zeros((c.rows, 8 * 128), device="cuda")
    out = torch.full_like(q, 7.0)
    ws = c.workspace(8)
    c.attend("f32", q, 7, 0.1, out, rc=-1)
    c.attend("f32", q, 8, float("nan"), out, rc=-1)
    c.attend("f32", q, 8, 0.1, out, workspace=ws[:-16], rc=-1 if ws.numel() > 16 else 0)
    if ws.numel() <= 16:
        out.fill_(7.0)
    c.max_length = c.stride * 64 + 1
    c.attend("f32", q, 8, 0.1, out, workspace=ws, rc=-1)
    assert (out == 7.0).all()


def test_a_decode_layer_to_token_logprobs(lib, torch, oracle):
    """A prompt block and decode steps as a layer runs them: the FP8 q/k/v projection,
    append with rotation, attention, the output projection with the residual, the
    final norm with the tied head, and the next tokens' log probabilities, against
    the same steps in 64 bits on the values that the cache holds."""
    from tests.tiling import ORDER_ROWS, tiled_bytes
    rng = np.random.default_rng(30)
    heads, group, dim, hidden, vocab, n, steps = 2, 2, 64, 256, 1000, 70, 3
    query = heads * group
    width = (query + 2 * heads) * dim
    table8 = np.array([oracle.fp8_decode(c) for c in range(256)], np.float64)

    def weight(rows, cols):
        codes = rng.integers(0, 256, (rows, cols)).astype(np.uint8)
        codes[(codes & 127) >= 0x70] &= 0x8F
        raw = torch.from_numpy(codes).cuda()
        dst = torch.empty(tiled_bytes(rows, cols), dtype=torch.uint8, device="cuda")
        assert lib.lunelette_cuda_tile_fp8(raw.data_ptr(), rows, cols, ORDER_ROWS, dst.data_ptr(),
                                           torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        return dst, table8[codes]

    (w_qkv, qkv64), (w_o, o64) = weight(width, hidden), weight(hidden, query * dim)
    s_qkv, s_o = 2.0 ** -6, 2.0 ** -6
    head = torch.randn((vocab, hidden), device="cuda").bfloat16()
    gain = torch.rand(hidden, device="cuda") + 0.5
    cos, sin, tables = rope_tables(torch, 256, dim)
    c = Cache(torch, [n], [n], heads, dim, max_length=256, stride=4, spare=3)
    c.table[0] = [3, 1, 0, 2]
    c.d_table.copy_(torch.from_numpy(c.table))
    stored = [np.zeros((0, heads, dim))] * 2
    stream = torch.cuda.current_stream().cuda_stream
    for step in range(1 + steps):
        count = n if step == 0 else 1
        length = n + step
        c.counts, c.lengths, c.rows, c.max_count = [count], [length], count, count
        c.offsets = np.array([0, count], np.int32)
        c.d_offsets.copy_(torch.from_numpy(c.offsets))
        c.d_lengths.fill_(length)
        x = rng.standard_normal((count, hidden)).astype(np.float32)
        d_x = torch.from_numpy(x).cuda()
        qkv = torch.empty((count, width), device="cuda")
        project = lib.lunelette_cuda_gemm_fp8 if count > 4 else lib.lunelette_cuda_gemv_fp8
        assert project(w_qkv.data_ptr(), width, hidden, s_qkv, d_x.data_ptr(), None, count, qkv.data_ptr(), stream) == 0
        q, k, v = qkv.split([query * dim, heads * dim, heads * dim], 1)
        q_out = torch.empty((count, query * dim), device="cuda")
        att = torch.empty((count, query * dim), device="cuda")
        c.append("f32", k, v, q, q_out, query, tables)
        c.attend("f32", q_out, query, dim ** -0.5, att)
        y = torch.empty((count, hidden), device="cuda")
        project = lib.lunelette_cuda_gemm_fp8 if count > 4 else lib.lunelette_cuda_gemv_fp8
        assert project(w_o.data_ptr(), hidden, query * dim, s_o, att.data_ptr(), d_x.data_ptr(), count, y.data_ptr(),
                       stream) == 0
        logits = torch.empty((1, vocab), device="cuda")
        flag = torch.zeros(1, dtype=torch.int32, device="cuda")
        assert lib.lunelette_cuda_head_bf16(head.data_ptr(), vocab, hidden, y[-1].data_ptr(), gain.data_ptr(),
                                            logits.data_ptr(), flag.data_ptr(), stream) == 0
        target = torch.tensor([step * 31 + 5], device="cuda")
        lp, ent = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda")
        ids, top = torch.zeros((1, 3), dtype=torch.int64, device="cuda"), torch.zeros((1, 3), device="cuda")
        assert lib.lunelette_cuda_token_logprobs(logits.data_ptr(), L.FLOAT32, 1, vocab, vocab, target.data_ptr(), 3,
                                                 lp.data_ptr(), ent.data_ptr(), ids.data_ptr(), top.data_ptr(),
                                                 stream) == 0
        torch.cuda.synchronize()
        # the same in 64 bits; the codes are decided on the projection's own FP32 output
        raw = qkv.double().cpu().numpy()
        want_qkv = (x.astype(np.float64) @ qkv64.T) * s_qkv
        qkv_size = (np.abs(x.astype(np.float64)) @ np.abs(qkv64).T) * s_qkv
        assert (np.abs(raw - want_qkv) <= 1e-5 * qkv_size).all()
        raw = raw.reshape(count, -1, dim)
        turned = np.zeros((count, query, dim))
        for i in range(count):
            p = length - count + i
            cp, sp = cos[p].astype(np.float64), sin[p].astype(np.float64)
            turned[i] = ref.rotate(raw[i, :query], cp, sp)
            for kind, r in ((0, ref.rotate(raw[i, query:query + heads], cp, sp)), (1, raw[i, query + heads:])):
                stored[kind] = np.concatenate([stored[kind], ref.dequantise(*ref.quantise(r))[None]])
        want, *size = ref.attention(turned, stored[0], stored[1], dim ** -0.5, length - count)
        # q_out is rounded to FP32 besides (2^-23 of each product)
        check_rows(torch, "f32", att.double().cpu().numpy().reshape(count, query, dim), want, 2 * size[0], *size[1:])
        a64 = att.double().cpu().numpy()
        y64 = a64[-1] @ (o64 * s_o).T + x[-1].astype(np.float64)
        y_size = np.abs(a64[-1]) @ np.abs(o64 * s_o).T + np.abs(x[-1])
        got_y = y[-1].double().cpu().numpy()
        assert (np.abs(got_y - y64) <= 1e-5 * y_size).all()
        h = head.double().cpu().numpy()
        normed = gain.double().cpu().numpy() * got_y / np.sqrt((got_y ** 2).mean() + 1e-5)
        logits64 = h @ normed
        e = 1e-5 * (np.abs(h) @ np.abs(normed)).max()  # the head's own bound
        m = logits64.max()
        logz = m + np.log(np.exp(logits64 - m).sum())
        assert abs(lp.item() - (logits64[target.item()] - logz)) <= 2 * e + 1e-5
        p = np.exp(logits64 - logz)
        assert abs(ent.item() + (p * np.log(p)).sum()) <= 2 * e * (1 + np.abs(np.log(p)).max()) + 1e-5
        order = np.argsort(-logits.cpu().numpy()[0], kind="stable")[:3]
        assert ids[0].tolist() == order.tolist()
        assert flag.item() == 0
    assert c.status.item() == 0
