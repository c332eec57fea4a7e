"""The 4-bit KV cache and the token log probabilities without a GPU: refused
arguments, the pool's layout, the roundings of the format and the search for a
row's sequence."""
import ctypes

import numpy as np
import pytest

import lunelette_b200 as L
from tests import kv4_reference as ref

A = 1 << 20  # a pointer that no call here follows: every call is refused or has no rows


def kv4(**change):
    f = dict(pool=A, layers=2, pages=9, kv_heads=3, head_dim=128)
    f.update(change)
    return L.Kv4(**f)


def rows(**change):
    f = dict(rows=0, sequences=2, offsets=A, lengths=A, page_tables=A, table_stride=4, max_count=5, max_length=256)
    f.update(change)
    return L.Rows(**f)


def append(lib, cache=None, r=None, **change):
    a = dict(layer=1, type=L.FLOAT32, k=A, k_stride=384, v=A, v_stride=400, q=A, q_stride=768, query_heads=6, q_out=A,
             q_out_stride=768, cos=A, sin=A, positions=256)
    a.update(change)
    return lib.lunelette_cuda_kv4_append(
        cache or kv4(), a["layer"], r or rows(), a["type"], a["k"], a["k_stride"], a["v"], a["v_stride"], a["q"],
        a["q_stride"], a["query_heads"], a["q_out"], a["q_out_stride"], a["cos"], a["sin"], a["positions"], None, None)


def read(lib, cache=None, r=None, **change):
    a = dict(layer=0, type=L.FLOAT16, k=A, k_stride=384, v=A, v_stride=384)
    a.update(change)
    return lib.lunelette_cuda_kv4_read(cache or kv4(), a["layer"], r or rows(), a["type"], a["k"], a["k_stride"], a["v"],
                                       a["v_stride"], None, None)


def attend(lib, cache=None, r=None, **change):
    a = dict(layer=0, type=L.BFLOAT16, q=A, q_stride=768, query_heads=6, scale=0.1, out=A, out_stride=768, ws=A,
             ws_bytes=1 << 40)
    a.update(change)
    return lib.lunelette_cuda_kv4_attention(cache or kv4(), a["layer"], r or rows(), a["type"], a["q"], a["q_stride"],
                                            a["query_heads"], a["scale"], a["out"], a["out_stride"], a["ws"],
                                            a["ws_bytes"], None, None)


BAD_CACHE = [dict(pool=None), dict(pool=A + 8), dict(layers=0), dict(pages=0), dict(pages=1 << 40), dict(kv_heads=0),
             dict(kv_heads=257), dict(head_dim=96), dict(head_dim=0)]
BAD_ROWS = [dict(rows=1 << 40), dict(sequences=1 << 40), dict(max_count=1 << 40), dict(max_length=1 << 40),
            dict(max_length=257), dict(offsets=A + 1), dict(lengths=A + 2), dict(page_tables=A + 3)]


def test_calls_without_rows_do_nothing(lib):
    assert append(lib) == read(lib) == attend(lib) == 0
    for r in (rows(sequences=0), rows(max_count=0), rows(offsets=None, lengths=None, page_tables=None)):
        assert append(lib, r=r) == read(lib, r=r) == attend(lib, r=r) == 0
    assert append(lib, k=None, v=None, q=None, q_out=None) == 0
    assert lib.lunelette_cuda_token_logprobs(None, L.FLOAT32, 0, 10, 10, None, 0, None, None, None, None, None) == 0


@pytest.mark.parametrize("call", [append, read, attend])
def test_bad_caches_and_rows_are_refused(lib, call):
    for change in BAD_CACHE:
        assert call(lib, cache=kv4(**change)) == -1, change
    for change in BAD_ROWS:
        assert call(lib, r=rows(**change)) == -1, change
    assert call(lib, layer=2) == -1
    assert call(lib, type=3) == -1 and call(lib, type=-1) == -1


def test_null_descriptors_are_refused(lib):
    null = [None, 0, rows(), 0, A, 384, A, 384]
    assert lib.lunelette_cuda_kv4_read(*null, None, None) == -1
    null[0], null[2] = kv4(), None
    assert lib.lunelette_cuda_kv4_read(*null, None, None) == -1
    assert lib.lunelette_cuda_kv4_attention_workspace(None, rows(), 6) == 0
    assert lib.lunelette_cuda_kv4_attention_workspace(kv4(), None, 6) == 0
    assert lib.lunelette_cuda_kv4_attention_workspace(kv4(), rows(), 7) == 0


@pytest.mark.parametrize("change", [
    dict(k_stride=383), dict(v_stride=383), dict(q_stride=767), dict(q_out_stride=767), dict(k=A + 2), dict(v=A + 1),
    dict(q=A + 3), dict(q_out=A + 2), dict(q=None), dict(q_out=None), dict(query_heads=0), dict(query_heads=5000),
    dict(cos=None), dict(sin=None), dict(cos=A + 4), dict(sin=A + 8), dict(positions=255), dict(k_stride=1 << 40)])
def test_append_refuses(lib, change):
    assert append(lib, **change) == -1


@pytest.mark.parametrize("change", [dict(k_stride=383), dict(v_stride=0), dict(k=A + 1), dict(v=A + 1)])
def test_read_refuses(lib, change):
    assert read(lib, **change) == -1


@pytest.mark.parametrize("change", [
    dict(q_stride=767), dict(out_stride=767), dict(q=A + 1), dict(out=A + 1), dict(query_heads=0), dict(query_heads=7),
    dict(query_heads=4098), dict(scale=float("nan")), dict(scale=float("inf")), dict(ws=A + 8)])
def test_attention_refuses(lib, change):
    assert attend(lib, **change) == -1


def test_attention_refuses_a_small_workspace(lib):
    r = rows(rows=5, max_length=256)
    need = lib.lunelette_cuda_kv4_attention_workspace(kv4(), r, 6)
    if need:
        assert attend(lib, r=r, ws_bytes=need - 1) == -1
        assert attend(lib, r=r, ws=None, ws_bytes=need) == -1


def test_logprobs_refuses(lib):
    def call(**change):
        a = dict(logits=A, type=L.BFLOAT16, rows=0, vocab=100, stride=100, targets=A, top=5, logprobs=A, entropy=A,
                 top_ids=A, top_logprobs=A)
        a.update(change)
        return lib.lunelette_cuda_token_logprobs(*a.values(), None)

    assert call() == 0
    for change in (dict(type=3), dict(vocab=0), dict(stride=99), dict(top=65), dict(vocab=4, stride=9), dict(targets=None),
                   dict(logprobs=None), dict(top_ids=None), dict(top_logprobs=None), dict(top=0), dict(logits=A + 1),
                   dict(rows=1 << 40), dict(vocab=1 << 40, stride=1 << 40), dict(targets=A + 4), dict(logprobs=A + 2),
                   dict(entropy=A + 1), dict(top_ids=A + 4), dict(top_logprobs=A + 2), dict(logits=None, rows=1)):
        assert call(**change) == -1, change


def test_pool_bytes(lib):
    for layers, pages, heads, dim in [(1, 1, 1, 64), (26, 1000, 8, 128), (2, 70000, 8, 128)]:
        assert lib.lunelette_cuda_kv4_bytes(layers, pages, heads, dim) == layers * pages * heads * ref.block_bytes(dim)
    assert lib.lunelette_cuda_kv4_bytes(1, 1, 1, 80) == 0
    assert lib.lunelette_cuda_kv4_bytes(0, 1, 1, 64) == 0


@pytest.mark.parametrize("dim", [64, 128])
def test_layout_covers_the_block_once_and_keeps_positions_apart(dim):
    owner = np.full(ref.block_bytes(dim), -1)
    for slot in range(64):
        even, group = np.arange(0, dim, 2), np.arange(dim // 32)
        at = np.concatenate([ref.k_byte(slot, even, dim), ref.v_byte(slot, even, dim)] +
                            [f(slot, group, dim) + i for f in (ref.k_scale_byte, ref.v_scale_byte) for i in (0, 1)])
        assert np.unique(at).size == at.size and (owner[at] == -1).all()
        owner[at] = slot
    assert (owner >= 0).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_fragment_reads_touch_each_bank_once(dim):
    """Lane (g, t) of the attention reads K chunk t of key g (dim / 8 bytes) and V
    chunk g of key 2 t (dim / 16 bytes): within each group of lanes that one
    shared-memory wavefront serves (128 bytes), every bank is hit once."""
    for name, chunk in (("k", dim // 8), ("v", dim // 16)):
        served = 128 // chunk  # lanes
        for key0 in range(0, 64, 16 if name == "v" else 8):
            for first in range(0, 32, served):
                banks = []
                for lane in range(first, first + served):
                    g, t = lane >> 2, lane & 3
                    if name == "k":
                        byte = (key0 + g) * (dim // 2) + t * chunk
                    else:
                        word = ref.v_byte(key0 + 2 * t, g * (dim // 8), dim) - ref.v_byte(0, 0, dim)
                        byte = word
                        # the lane's words are consecutive
                        last = ref.v_byte(key0 + 2 * t, (g + 1) * (dim // 8) - 1, dim) - ref.v_byte(0, 0, dim)
                        assert last == byte + chunk - 1
                    banks += [(byte // 4 + i) % 32 for i in range(chunk // 4)]
                assert sorted(banks) == list(range(32)), (name, key0, first)


def test_stored_values_are_exact_in_fp16():
    rng = np.random.default_rng(3)
    m = np.concatenate([rng.standard_normal(4000) * np.exp2(rng.integers(-30, 20, 4000)), [0.0, 1e30, -1e30, 65280.0]])
    d = ref.scale_of(m)
    assert np.array_equal(d, d.astype(np.float16).astype(np.float64))
    for c in range(-8, 8):
        assert np.array_equal(d * c, (d * c).astype(np.float16).astype(np.float64))
    # and in one FP16 fused multiply-add from 16 + c: the addend -24 d is representable
    ok = np.abs(24 * d) < 65504
    assert np.array_equal(24 * d[ok], (24 * d[ok]).astype(np.float16).astype(np.float64))


def find_sequence(offsets, row):
    """kv4_sequence_of_row of kv4.cuh, lane by lane."""
    lo, n = 0, len(offsets) - 1
    while n > 32:
        step = (n + 31) // 32
        before = [lane * step < n and (lane == 0 or offsets[lo + lane * step] <= row) for lane in range(32)]
        last = max(i for i in range(32) if before[i])
        lo += last * step
        n = min(step, n - last * step)
    return lo + max(i for i in range(n) if i == 0 or offsets[lo + i] <= row)


def test_row_search_finds_the_sequence_that_holds_the_row():
    rng = np.random.default_rng(4)
    for n in (1, 2, 5, 31, 32, 33, 64, 100, 1000, 1025, 3000):
        counts = rng.integers(0, 4, n) * rng.integers(0, 2, n)
        counts[rng.integers(n)] += 3
        offsets = np.concatenate([[0], np.cumsum(counts)])
        for row in np.unique(np.clip(np.concatenate([offsets, offsets - 1, offsets + 1]), 0, offsets[-1] - 1)):
            s = find_sequence(offsets, row)
            assert offsets[s] <= row < offsets[s + 1]


def test_quantisation_error_is_at_most_half_a_step_inside_and_one_at_the_far_end():
    rng = np.random.default_rng(5)
    r = rng.standard_normal((500, 32)) * np.exp2(rng.integers(-6, 7, (500, 1)))
    codes, d = ref.quantise(r)
    # the far sign's extreme is clipped at 7 steps where |r| may reach 8 and d is off by 2^-9 of itself
    assert (np.abs(ref.dequantise(codes, d) - r) <= np.abs(d) * (1 + 8 * 2.0 ** -8)).all()
    inside = np.abs(r) <= 7.4 * np.abs(d)
    assert (np.abs(ref.dequantise(codes, d) - r)[inside] <= 0.5 * np.broadcast_to(np.abs(d), r.shape)[inside]).all()


def test_values_from_subnormal_codes_are_exact_in_fp16():
    """The decode kernel's conversion: a code alone in a half's bits 0..3 or 4..7 is the subnormal c 2^-24 or
    c 2^-20; one multiply-add with d 2^15 or d 2^11 and -d 2^-6 leaves d (c - 8) 2^-9. Every operand and the result
    is an FP16 for 2^-8 <= |d| < 2; elsewhere c - 8, from a half of 1024 + c or 1024 + 16 c, is multiplied by d."""
    def exact(x):
        with np.errstate(over="ignore"):
            return np.array_equal(x, x.astype(np.float16).astype(np.float64))

    every = (np.arange(128, 256)[:, None] * np.exp2(np.arange(-15.0, -6.0))[None]).reshape(-1)
    every = np.concatenate([every, -every])[:, None]
    assert np.abs(every).min() == 2.0 ** -8 and np.abs(every).max() < 2.0
    c = np.arange(16.0)[None]
    for shift, factor in ((24, 15), (20, 11)):
        code = c * 2.0 ** -shift
        bits = (np.arange(16, dtype=np.uint16) << (24 - shift)).view(np.float16).astype(np.float64)
        assert np.array_equal(code[0], bits)
        assert exact(every * 2.0 ** factor) and exact(-every * 2.0 ** -6)
        value = code * (every * 2.0 ** factor) - every * 2.0 ** -6
        assert np.array_equal(value, every * (c - 8) * 2.0 ** -9) and exact(value)
    # just outside: a result below FP16's last step, a factor past its largest value
    assert not exact(np.array([[129 * 2.0 ** -16]]) * (c - 8) * 2.0 ** -9)
    assert not exact(np.array([2.0 * 2.0 ** 15]))
    codes = np.arange(16, dtype=np.uint16)
    low, high = ((0x6400 | codes << s).astype(np.uint16).view(np.float16).astype(np.float64) for s in (0, 4))
    assert np.array_equal(low - 1032, codes - 8.0) and np.array_equal(high / 16 - 72, codes - 8.0)
    assert np.array_equal(np.array([0x6408, 0x2c00, 0xd480], np.uint16).view(np.float16), [1032, 1 / 16, -72])
