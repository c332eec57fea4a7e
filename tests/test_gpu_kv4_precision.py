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
