"""The upper end of the 4-bit cache's range: finite bf16 rows stay finite (write, read-back, attention in place).

The block exponent e is held at 125: 6 x 2^125 = 1.5 x 2^127 is the largest value that bf16 and fp32 hold and a block can
stand for (the next code's, 2^128, is an infinity there).  A block whose largest magnitude is at least 1.75 x 2^127 would
round to that infinity; its largest values become 1.5 x 2^127 instead."""
import numpy as np
import pytest
import torch

from vllm_trianglemix_amd import ops

gpu = pytest.mark.gpu
DEV = "cuda:0"
TOP = 1.5 * 2.0 ** 127
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def stored(x):
    """What blocks ``[..., 32]`` with magnitudes from 3.5 x 2^125 on stand for: the nearest of the grid times 2^125, ties to
    the even code, everything past 5 x 2^125 its largest value."""
    y = np.abs(x) / 2.0 ** 125
    d = np.abs(y[..., None] - GRID)
    code = np.where(d == d.min(-1, keepdims=True), np.arange(8) % 2, 2).argmin(-1)
    return np.copysign(GRID[code] * 2.0 ** 125, x)


def near_the_top(rng, blocks):
    """bf16 rows: a largest magnitude between 3.5 x 2^125 and the type's largest value, the others from zero to it."""
    x = rng.uniform(0, 1, (blocks, 32)) ** 3 * rng.uniform(3.5, 8, (blocks, 1)) * rng.choice([-1.0, 1.0], (blocks, 32))
    top = np.array([3.5, 6.0, 6.96875, 7.0, 7.03125, 7.5, 7.96875])  # (multiples of bf16's step there)
    x[:, 5] = np.where(np.arange(blocks) < 14, np.tile(top, 8)[:blocks] * np.where(np.arange(blocks) % 2, -1, 1), x[:, 5])
    x[np.abs(x) > 7.96875] = 7.96875
    t = torch.from_numpy(x * 2.0 ** 125).to(torch.bfloat16)
    amax = t.double().abs().amax(1)
    t[:, 9] = torch.where(amax < 3.5 * 2.0 ** 125, torch.full_like(t[:, 9], 3.5 * 2.0 ** 125), t[:, 9])
    return t


def caches_of(rows_k, rows_v, heads, dim, page):
    n = rows_k.shape[0]
    pages = -(-n // page)
    caches = [torch.zeros(ops.fp4_cache_shape(pages, page, heads, dim), dtype=torch.uint8, device=DEV) for _ in range(2)]
    ops.reshape_and_cache_fp4(rows_k.to(DEV), rows_v.to(DEV), *caches, torch.arange(n, device=DEV))
    table = torch.arange(pages, dtype=torch.int32, device=DEV).view(1, -1)
    return caches, table, torch.tensor([n], dtype=torch.int32, device=DEV)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_near_the_largest_bf16_value_stay_finite(dim):
    rng = np.random.default_rng(dim)
    n, heads = 7, 2
    x = near_the_top(rng, n * heads * dim // 32)
    rows = x.view(n, heads, dim)
    want = stored(x.double().numpy()).reshape(n, heads, dim)
    assert np.isfinite(x.double().numpy()).all() and np.abs(want).max() == TOP
    caches, table, lens = caches_of(rows, -rows, heads, dim, 16)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    k, v = ops.gather_dequant_kv_fp4(*caches, table, lens, zero, n, n, torch.bfloat16)
    assert np.array_equal(k.double().cpu().numpy(), want) and np.array_equal(v.double().cpu().numpy(), -want)
    k, v = ops.gather_dequant_kv_fp4(*caches, table, lens, zero, n, n, torch.float16)
    assert np.array_equal(k.double().cpu().numpy(), np.clip(want, -65504, 65504))
    # the scale bytes themselves: e = 125
    nb = heads * 16 * dim // 2
    for c in caches:
        scales = c.view(1, -1)[0, nb:].view(heads, dim // 32, 16)[:, :, :n]
        assert (scales == 252).all()


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_over_the_largest_values(dim, dtype):
    """Two positions, keys of zeros (equal weights): the first row sees ones, the second the mean of 1 and the largest value,
    (1 + 1.5 x 2^127) / 2, which is 0.75 x 2^127 in fp32."""
    big = torch.finfo(torch.bfloat16).max
    v = torch.ones(2, 1, dim, dtype=torch.bfloat16)
    v[1] = big
    v[1, 0, 1::2] = -big
    sign = torch.ones(dim, device=DEV)
    sign[1::2] = -1
    for heads in (1, 4, 16):
        caches, table, lens = caches_of(torch.zeros_like(v), v, 1, dim, 16)
        q = torch.ones(2, heads, dim, dtype=dtype, device=DEV)
        out = torch.zeros(2, heads, dim, device=DEV)
        ws = ops.decode_fp4_workspace(1, 2, heads, 1, dim, DEV)
        ops.decode_attention_fp4(q, *caches, out, table, lens, 0.1, ws, rows_per_request=2)
        assert (out[0] == 1).all()
        assert torch.equal(out[1], (0.5 * TOP * sign).expand(heads, dim))


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_keys_of_the_largest_values_give_finite_scores(dim):
    """Scores of 2^127 scaled down are finite numbers: the key with the larger one gets all the weight."""
    k = torch.zeros(2, 1, dim, dtype=torch.bfloat16)
    k[0, 0, 3], k[1, 0, 3] = torch.finfo(torch.bfloat16).max, 1.0
    v = torch.ones(2, 1, dim, dtype=torch.bfloat16)
    v[1] = 4
    caches, table, lens = caches_of(k, v, 1, dim, 16)
    q = torch.zeros(1, 2, dim, dtype=torch.bfloat16, device=DEV)
    q[0, 0, 3], q[0, 1, 3] = 1.0, -1.0
    out = torch.zeros(1, 2, dim, device=DEV)
    ops.decode_attention_fp4(q, *caches, out, table, lens, 2.0 ** -100, ops.decode_fp4_workspace(1, 1, 2, 1, dim, DEV))
    assert (out[0, 0] == 1).all() and (out[0, 1] == 4).all()
