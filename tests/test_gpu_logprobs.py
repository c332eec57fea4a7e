"""Token log probabilities, entropy and top alternatives on the GPU against the
definition in 64 bits."""
import numpy as np
import pytest

import lunelette_b200 as L

pytestmark = pytest.mark.gpu

TYPES = {"f32": (L.FLOAT32, "float32"), "bf16": (L.BFLOAT16, "bfloat16"), "f16": (L.FLOAT16, "float16")}


@pytest.fixture(scope="module")
def torch():
    import torch
    torch.cuda.init()
    return torch


def call(torch, name, logits, targets=None, top=0, entropy=True, rc=0):
    rows, vocab = logits.shape
    lp = torch.full((rows,), 7.0, device="cuda") if targets is not None else None
    ent = torch.full((rows,), 7.0, device="cuda") if entropy else None
    ids = torch.full((rows, top), -7, dtype=torch.int64, device="cuda") if top else None
    tlp = torch.full((rows, top), 7.0, device="cuda") if top else None
    stride = logits.stride(0) if rows > 1 else vocab
    p = [x.data_ptr() if x is not None else None for x in (lp, ent, ids, tlp)]
    assert L.library().lunelette_cuda_token_logprobs(
        logits.data_ptr(), TYPES[name][0], rows, vocab, stride, targets.data_ptr() if targets is not None else None,
        top, *p, torch.cuda.current_stream().cuda_stream) == rc
    torch.cuda.synchronize()
    return [x.cpu().numpy() if x is not None else None for x in (lp, ent, ids, tlp)]


def check(torch, name, logits, top, seed=0):
    rows, vocab = logits.shape
    rng = np.random.default_rng(seed)
    targets = torch.from_numpy(rng.integers(0, vocab, rows)).cuda()
    lp, ent, ids, tlp = call(torch, name, logits, targets, top)
    x = logits.double().cpu().numpy()
    t = targets.cpu().numpy()
    for r in range(rows):
        m = x[r].max()
        e = np.exp(x[r] - m)
        z = e.sum()
        want = x[r] - m - np.log(z)
        p = e / z
        live = p > 0
        # x - m is rounded once (2^-24), ln Z carries the relative error of Z: the exponentials' (2^-22 and
        # 2^-23 of their argument, whose weighted mean is the entropy's size) and the sum's
        span = (p[live] * np.abs(x[r][live] - m)).sum()
        ez = 2.0 ** -21 + 2.0 ** -22 * span
        # the largest values' sums: at most 2^-24 per addition over the chain of a thread and the tree
        ez += 2.0 ** -24 * 64

        def bound(v):
            return ez + 2.0 ** -23 * (np.abs(v) + np.abs(np.log(z)))

        assert lp[r] == want[t[r]] or abs(lp[r] - want[t[r]]) <= bound(want[t[r]]), (r, lp[r], want[t[r]])
        h = -(p[live] * want[live]).sum()
        assert abs(ent[r] - h) <= ez * (2 + span) + 2.0 ** -22 * (h + span), (r, ent[r], h)
        if top:
            order = np.argsort(-x[r], kind="stable")[:top]
            assert ids[r].tolist() == order.tolist(), r
            w = want[order]
            same = (tlp[r] == w) | (np.abs(tlp[r] - np.where(np.isinf(w), 0, w)) <= bound(np.where(np.isinf(w), 0, w)))
            assert same.all(), r


def make(torch, name, rows, vocab, pad=0, seed=0, scale=2.5, offset=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = torch.randn((rows, vocab + pad + offset), generator=gen, device="cuda") * scale
    return x.to(getattr(torch, TYPES[name][1]))[:, offset:offset + vocab]


@pytest.mark.parametrize("name,rows,vocab,top,pad,offset", [
    ("f32", 1, 1, 1, 0, 0), ("f32", 3, 2, 2, 0, 0), ("f32", 1, 131072, 5, 0, 0), ("f32", 5, 131072, 64, 0, 0),
    ("f32", 300, 1000, 20, 3, 0), ("bf16", 7, 50001, 8, 2, 0), ("bf16", 3, 131072, 20, 0, 0), ("f16", 2, 4097, 33, 5, 1),
    ("bf16", 1, 40, 40, 0, 0), ("f32", 2, 64, 64, 0, 0), ("f32", 700, 333, 0, 0, 0), ("f16", 40, 30000, 1, 1, 3),
    ("f32", 1200, 257, 64, 1, 1), ("bf16", 160, 20011, 64, 0, 0), ("f32", 30, 9000, 7, 0, 0)])
def test_matches_definition(torch, name, rows, vocab, top, pad, offset):
    check(torch, name, make(torch, name, rows, vocab, pad, rows + vocab, offset=offset), top)


@pytest.mark.parametrize("kind", ["ascending", "descending", "constant", "sawtooth", "peaks", "wide"])
@pytest.mark.parametrize("rows,vocab", [(2, 70000), (200, 5000)])
def test_orders_that_defeat_a_threshold(torch, kind, rows, vocab):
    """Rows in which every element beats those before it, all are equal, or few dominate."""
    i = np.arange(vocab)
    x = {"ascending": i * 1e-3, "descending": -i * 1e-3, "constant": np.zeros(vocab), "sawtooth": (i * 37 % 101) * 0.05,
         "peaks": np.where(i % 9973 == 5, 30.0 + i * 1e-4, 0.0), "wide": (i * 7919 % vocab) * 2e-3 - 80.0}[kind]
    x = np.stack([np.roll(x, 13 * r) for r in range(rows)]).astype(np.float32)
    check(torch, "f32", torch.from_numpy(x).cuda(), 33)


def test_masked_vocabulary(torch):
    x = make(torch, "f32", 6, 3000, seed=4)
    x[0, 10:] = -np.inf                       # ten left
    x[1, :2990] = -np.inf
    x[2, 1:] = -np.inf                        # one left
    x[3] = torch.finfo(torch.float32).min     # the type's lowest value: a uniform row
    x[4, ::2] = torch.finfo(torch.float32).min
    check(torch, "f32", x, 20)
    lp, ent, ids, tlp = call(torch, "f32", x, torch.full((6,), 2999, device="cuda"), 20)
    assert lp[0] == -np.inf and lp[2] == -np.inf and ent[2] == 0.0
    assert ids[2].tolist() == list(range(20)) and tlp[2, 0] == 0.0 and (tlp[2, 1:] == -np.inf).all()


def test_rows_without_a_distribution(torch):
    for rows, vocab in ((5, 3000), (5, 100000), (400, 500)):
        x = make(torch, "f32", rows, vocab, seed=5)
        x[0, 77] = float("nan")
        x[1, 78] = float("inf")
        x[2] = -float("inf")
        x[3, 79], x[3, 5] = float("nan"), float("inf")
        lp, ent, ids, tlp = call(torch, "f32", x, torch.zeros(rows, dtype=torch.int64, device="cuda"), 3)
        assert np.isnan(lp[:4]).all() and np.isnan(ent[:4]).all() and np.isnan(tlp[:4]).all()
        assert np.isfinite(lp[4:]).all() and np.isfinite(ent[4:]).all()
        assert ids[0, 0] == 77 and ids[1, 0] == 78 and ids[2].tolist() == [0, 1, 2] and ids[3, :2].tolist() == [79, 5]


def test_targets_outside_the_vocabulary(torch):
    x = make(torch, "bf16", 4, 90, seed=6)
    lp, ent, _, _ = call(torch, "bf16", x, torch.tensor([-1, 90, 1 << 40, 89], device="cuda"))
    assert np.isnan(lp[:3]).all() and np.isfinite(lp[3]) and np.isfinite(ent).all()


def test_outputs_may_be_left_out(torch):
    x = make(torch, "f32", 9, 5000, seed=7)
    targets = torch.arange(9, device="cuda")
    full = call(torch, "f32", x, targets, 4)
    assert np.array_equal(call(torch, "f32", x, targets, 0, entropy=False)[0], full[0])
    assert np.array_equal(call(torch, "f32", x, None, 0)[1], full[1])
    got = call(torch, "f32", x, None, 4, entropy=False)
    assert np.array_equal(got[2], full[2]) and np.array_equal(got[3], full[3])


def test_signed_zeros_tie(torch):
    x = torch.full((1, 300), -1.0, device="cuda")
    x[0, 100], x[0, 200] = -0.0, 0.0
    assert call(torch, "f32", x, None, 2)[2].tolist() == [[100, 200]]


def test_same_bits_every_time_and_in_a_graph(torch):
    for name, rows, vocab in (("f32", 1, 131072), ("bf16", 333, 7001)):
        x = make(torch, name, rows, vocab, seed=8)
        targets = torch.zeros(rows, dtype=torch.int64, device="cuda")
        first = call(torch, name, x, targets, 17)
        for _ in range(5):
            assert all(np.array_equal(a, b) for a, b in zip(first, call(torch, name, x, targets, 17)))
        out = [torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"),
               torch.zeros((rows, 17), dtype=torch.int64, device="cuda"), torch.zeros((rows, 17), device="cuda")]
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            assert L.library().lunelette_cuda_token_logprobs(
                x.data_ptr(), TYPES[name][0], rows, vocab, x.stride(0), targets.data_ptr(), 17,
                *(o.data_ptr() for o in out), torch.cuda.current_stream().cuda_stream) == 0
        graph.replay()
        torch.cuda.synchronize()
        assert all(np.array_equal(a, b.cpu().numpy()) for a, b in zip(first, out))


@pytest.mark.parametrize("name,rows,vocab", [("f32", 1, 131072), ("f32", 40, 131072), ("bf16", 3, 50001)])
@pytest.mark.parametrize("left", [0, 1, 3, 40])
def test_few_adjacent_tokens_left_by_a_mask(torch, name, rows, vocab, left):
    """A grammar that allows digits, say: fewer tokens than `top`, next to each other, in rows of many blocks."""
    x = make(torch, name, rows, vocab, seed=9).clone()
    keep = x[:, 700:700 + left].clone()
    x[:] = -np.inf
    x[:, 700:700 + left] = keep
    if left:
        check(torch, name, x, 20)
    lp, ent, ids, tlp = call(torch, name, x, torch.full((rows,), 700, device="cuda"), 20)
    order = np.sort(ids, 1)
    rest = np.arange(20 - min(left, 20))
    assert (order[:, :rest.size] == rest).all() and ((order[:, rest.size:] >= 700) & (order[:, rest.size:] < 700 + left)).all()
    assert np.isnan(lp).all() == (left == 0) and np.isfinite(lp).all() == (left > 0)
