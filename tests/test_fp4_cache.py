"""The 4-bit (MXFP4) paged K/V cache: write, read-back and attention in place, against the format and the formulas in 64
bits (tests/fp4_reference.py).  The write is exact, so it is compared byte for byte; attention outputs to a bound derived
from their roundings (``fp4_reference.bound``)."""
import ctypes

import numpy as np
import pytest
import torch

import fp4_reference as ref
from vllm_trianglemix_amd import _lib, ops

gpu = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


# ------------------------------------------------------------------------------------------------ without a GPU
def test_reference_format_round_trips():
    rng = np.random.default_rng(0)
    for dim in (64, 128):
        for is_v in (False, True):
            codes = rng.integers(0, 16, (3, 16, 2, dim)).astype(np.uint8)
            scales = rng.integers(1, 254, (3, 16, 2, dim // 32)).astype(np.uint8)
            raw = ref.pack(codes, scales, is_v)
            assert raw.shape[1] == np.prod(ops.fp4_cache_shape(3, 16, 2, dim)[1:])
            assert np.array_equal(ref.unpack(raw, 2, dim, 16, is_v), ref.values(codes, scales))
    x = rng.standard_normal((5, 64)) * np.ldexp(1.0, rng.integers(-20, 20, (5, 1)))
    c, s = ref.quantise(x)
    y = ref.values(c, s)
    # half a step of the top binade is 2^e, and amax >= 3.5 x 2^e
    assert (np.abs(x - y).reshape(5, 2, 32) <= np.abs(x).reshape(5, 2, 32).max(-1, keepdims=True) / 3.5).all()
    c2, s2 = ref.quantise(y)
    assert np.array_equal(ref.values(c2, s2), y)  # its own values are fixed points


def test_cache_shape_refusals():
    assert ops.fp4_cache_shape(7, 32, 8, 128) == (7, 32, 8, 68)
    for bad in ((4, 16, 8, 96), (4, 8, 8, 128), (4, 24, 8, 128)):
        with pytest.raises(RuntimeError):
            ops.fp4_cache_shape(*bad)


def test_decode_struct_has_the_headers_size():
    import os
    import subprocess
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "s.c"), os.path.join(d, "s")
        with open(c, "w") as f:
            f.write('#include <stdio.h>\n#include "trianglemix_hip.h"\nint main(void){printf("%zu", sizeof(tmx_decode_fp4_args_t));return 0;}\n')
        subprocess.run(["gcc", "-I", os.path.join(root, "include"), c, "-o", exe], check=True)
        assert int(subprocess.run([exe], check=True, capture_output=True, text=True).stdout) == ctypes.sizeof(_lib.DecodeFp4Args)


def _args(**kw):
    """A well-formed argument block over made-up, aligned addresses (calls with it are refused before any launch)."""
    a = _lib.DecodeFp4Args()
    a.struct_size, a.io_dtype, a.out_dtype, a.scale = ctypes.sizeof(a), _lib.TMX_BF16, _lib.TMX_BF16, 0.1
    a.batch, a.rows_per_request, a.num_heads, a.num_kv_heads, a.head_dim, a.page_size = 2, 1, 8, 2, 128, 16
    a.out = a.q = a.k = a.v = a.block_table = a.seq_lens = a.partial_o = a.partial_ml = 4096
    a.out_stride_t = a.q_stride_t = 8 * 128
    a.out_stride_h = a.q_stride_h = 128
    a.kv_stride_page, a.num_pages, a.block_table_stride, a.max_blocks = 16 * 2 * 68, 9, 4, 4
    a.workspace_rows = 1 << 40
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change, code", [
    (dict(struct_size=8), _lib.TMX_ERR_INVALID_ARG), (dict(io_dtype=_lib.TMX_F32), _lib.TMX_ERR_UNSUPPORTED),
    (dict(out_dtype=_lib.TMX_F16), _lib.TMX_ERR_UNSUPPORTED), (dict(head_dim=96), _lib.TMX_ERR_UNSUPPORTED),
    (dict(num_heads=7), _lib.TMX_ERR_INVALID_ARG), (dict(rows_per_request=0), _lib.TMX_ERR_INVALID_ARG),
    (dict(rows_per_request=17), _lib.TMX_ERR_UNSUPPORTED), (dict(rows_per_request=2 ** 31 - 1), _lib.TMX_ERR_UNSUPPORTED),
    (dict(scale=0.0), _lib.TMX_ERR_INVALID_ARG), (dict(scale=float("nan")), _lib.TMX_ERR_INVALID_ARG),
    (dict(page_size=24), _lib.TMX_ERR_UNSUPPORTED), (dict(page_size=8), _lib.TMX_ERR_UNSUPPORTED),
    (dict(q=None), _lib.TMX_ERR_INVALID_ARG), (dict(num_pages=0), _lib.TMX_ERR_INVALID_ARG),
    (dict(kv_stride_page=16 * 2 * 68 - 16), _lib.TMX_ERR_INVALID_ARG), (dict(kv_stride_page=16 * 2 * 68 + 8), _lib.TMX_ERR_INVALID_ARG),
    (dict(k=4104), _lib.TMX_ERR_INVALID_ARG), (dict(q_stride_h=132), _lib.TMX_ERR_INVALID_ARG),
    (dict(max_blocks=-1), _lib.TMX_ERR_INVALID_ARG), (dict(batch=-1), _lib.TMX_ERR_INVALID_ARG),
    (dict(batch=70000), _lib.TMX_ERR_UNSUPPORTED), (dict(num_heads=2048, num_kv_heads=1024, page_size=1 << 20), _lib.TMX_ERR_UNSUPPORTED),
    (dict(max_blocks=2 ** 31 - 1), _lib.TMX_ERR_UNSUPPORTED), (dict(batch=60000, max_blocks=1 << 20), _lib.TMX_ERR_UNSUPPORTED),
    (dict(workspace_rows=1 << 4), None),
])
def test_decode_refuses_bad_arguments(change, code):
    lib = _lib.load()
    got = lib.tmx_decode_attention_fp4(ctypes.byref(_args(**change)), None)
    # (too small a work area shows once the chip's size is known; without a chip that is an error of its own)
    assert got == code if code is not None else got in (_lib.TMX_ERR_INVALID_ARG, _lib.TMX_ERR_HIP)
    assert lib.tmx_last_error()


def test_decode_of_an_empty_batch_is_nothing():
    assert _lib.load().tmx_decode_attention_fp4(ctypes.byref(_args(batch=0, q=None)), None) == _lib.TMX_OK
    assert _lib.load().tmx_decode_attention_fp4(None, None) == _lib.TMX_ERR_INVALID_ARG
    assert _lib.load().tmx_decode_fp4_workspace_rows(0, 1, 8, 2, 128, 256) == 0
    assert _lib.load().tmx_decode_fp4_workspace_rows(3, 2, 8, 2, 128, 256) >= 3 * 2 * 8


@pytest.mark.parametrize("change, code", [
    (dict(dim=96), _lib.TMX_ERR_UNSUPPORTED), (dict(dtype=_lib.TMX_F32), _lib.TMX_ERR_UNSUPPORTED),
    (dict(page=17), _lib.TMX_ERR_UNSUPPORTED), (dict(tokens=-1), _lib.TMX_ERR_INVALID_ARG), (dict(ptr=4104), _lib.TMX_ERR_INVALID_ARG),
    (dict(stride=4), _lib.TMX_ERR_INVALID_ARG), (dict(page_stride=64), _lib.TMX_ERR_INVALID_ARG), (dict(ptr=None), _lib.TMX_ERR_INVALID_ARG),
    (dict(heads=0), _lib.TMX_ERR_INVALID_ARG),
])
def test_write_and_gather_refuse_bad_arguments(change, code):
    c = dict(dim=128, dtype=_lib.TMX_BF16, page=16, tokens=4, ptr=4096, stride=128, page_stride=16 * 2 * 68, heads=2, pages=9)
    c.update(change)
    lib = _lib.load()
    assert lib.tmx_reshape_and_cache_fp4(c["ptr"], c["ptr"], c["stride"], c["stride"], c["stride"], c["stride"], c["ptr"],
                                         c["ptr"], c["page_stride"], c["pages"], c["ptr"], c["tokens"], c["heads"], c["dim"],
                                         c["page"], c["dtype"], None) == code
    if "stride" in change:
        return
    assert lib.tmx_gather_dequant_kv_fp4(c["ptr"], c["ptr"], c["page_stride"], c["pages"], c["ptr"], 4, 4, c["page"], c["ptr"],
                                         c["ptr"], 2, c["tokens"], c["heads"], c["dim"], c["ptr"], c["ptr"], 100, c["dtype"],
                                         None) == code


def test_tensors_on_the_cpu_are_refused():
    k = torch.zeros(ops.fp4_cache_shape(4, 16, 2, 64), dtype=torch.uint8)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.reshape_and_cache_fp4(x, x, k, k, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.gather_dequant_kv_fp4(k, k, torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
                                  torch.zeros(1, dtype=torch.int32), 1, 1, torch.bfloat16)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.decode_attention_fp4(x, k, k, x, torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32), 1.0, (x, x))


# ------------------------------------------------------------------------------------------------ on the GPU
def _values_of(rng, shape, dtype):
    """Rows over many magnitudes, with zeros, ties between codes and (fp16 / bf16) subnormals."""
    x = rng.standard_normal(shape) * np.ldexp(1.0, rng.integers(-6, 7, (*shape[:-1], 1)))
    x[rng.random(shape) < 0.05] = 0.0
    grid = rng.choice(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.99, 7.0]), shape)
    x = np.where(rng.random(shape) < 0.2, grid, x)
    x.reshape(-1, 32)[::7] = 0.0
    x.reshape(-1, 32)[1::11] *= 2.0 ** (-24 if dtype == torch.float16 else -130)
    if dtype == torch.float16:
        x.reshape(-1, 32)[2::13] *= 2.0 ** 10
        x = np.clip(x, -65504, 65504)
    return torch.from_numpy(x).to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim, heads, page", [(128, 2, 16), (64, 3, 16), (128, 1, 64), (64, 8, 32), (128, 8, 16)])
@pytest.mark.parametrize("tokens", [1, 5, 77])
def test_write_stores_the_formats_bytes(dtype, dim, heads, page, tokens):
    rng = np.random.default_rng(tokens * 1000 + dim + heads)
    pages = -(-tokens // page) + 3
    shape = ops.fp4_cache_shape(pages, page, heads, dim)
    # rows as slices of a fused projection (a row stride of their own), K and V apart
    qkv = torch.zeros(tokens, 3, heads, dim, dtype=dtype)
    qkv[:, 1], qkv[:, 2] = _values_of(rng, (tokens, heads, dim), dtype), _values_of(rng, (tokens, heads, dim), dtype)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    if tokens > 4:
        slots[1], slots[3], slots[4] = -1, pages * page, 2 ** 62  # padding, and slots the cache does not have
    start = rng.integers(0, 256, (2, *shape)).astype(np.uint8)
    caches = [torch.from_numpy(s.copy()).to(DEV) for s in start]
    d = qkv.to(DEV)
    ops.reshape_and_cache_fp4(d[:, 1], d[:, 2], caches[0], caches[1], torch.from_numpy(slots).to(DEV))
    for x in range(2):
        rows = qkv[:, 1 + x].double().numpy()
        want = start[x].reshape(pages, -1).copy()
        full = np.zeros((pages, page, heads, dim), np.uint8), np.zeros((pages, page, heads, dim // 32), np.uint8)
        mine = np.zeros((pages, page), bool)
        codes, scales = ref.quantise(rows)
        for t, s in enumerate(slots):
            if 0 <= s < pages * page:
                full[0][s // page, s % page], full[1][s // page, s % page] = codes[t], scales[t]
                mine[s // page, s % page] = True
        packed = ref.pack(*full, x == 1)
        mask = ref.pack(np.where(mine[..., None, None], 15, 0).astype(np.uint8) + 0 * full[0],
                        np.where(mine[..., None, None], 255, 0).astype(np.uint8) + 0 * full[1], x == 1)
        want = (want & ~mask) | (packed & mask)
        assert np.array_equal(caches[x].cpu().numpy().reshape(pages, -1), want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_blocks_with_infinities_and_nans_read_as_nan(dtype):
    x = torch.ones(4, 1, 64, dtype=dtype)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 0] = float("inf"), float("nan"), -float("inf")
    caches = [torch.zeros(ops.fp4_cache_shape(1, 16, 1, 64), dtype=torch.uint8, device=DEV) for _ in range(2)]
    ops.reshape_and_cache_fp4(x.to(DEV), x.to(DEV), *caches, torch.arange(4, device=DEV))
    k, v = ops.gather_dequant_kv_fp4(*caches, torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([4], dtype=torch.int32, device=DEV),
                                     torch.zeros(2, dtype=torch.int32, device=DEV), 4, 4, dtype)
    for got in (k.cpu(), v.cpu()):
        nan = torch.isnan(got[:, 0].float())
        assert nan[0].tolist() == [True] * 32 + [False] * 32 and nan[1].tolist() == [False] * 32 + [True] * 32
        assert nan[2].tolist() == [True] * 32 + [False] * 32 and not nan[3].any()
        assert (got[:, 0][~nan] == 1).all()


class Batch:
    """Sequences of given lengths with scattered pages of a cache made of random rows (quantised on the host)."""

    def __init__(self, seed, lens, heads, kv_heads, dim, page, m=1, spare=2, page_gap=0):
        rng = np.random.default_rng(seed)
        self.lens, self.H, self.Hkv, self.D, self.page, self.m = lens, heads, kv_heads, dim, page, m
        need = [max(0, -(-n // page)) for n in lens]
        pages = max(1, sum(need) + spare)
        order = rng.permutation(pages)
        self.table = np.full((len(lens), max(need + [1]) + 1), -1, np.int32)
        at = 0
        for b, c in enumerate(need):
            self.table[b, :c] = order[at:at + c]
            at += c
        self.raw = []
        for is_v in (False, True):
            rows = rng.standard_normal((pages, page, kv_heads, dim))
            rows[..., ::29] *= 4
            self.raw.append(ref.pack(*ref.quantise(rows), is_v))
        # a page stride of its own: the caches are views into a larger allocation
        size = self.raw[0].shape[1]
        self.caches = []
        for raw in self.raw:
            big = torch.full((pages, size + page_gap), 255, dtype=torch.uint8, device=DEV)
            view = big.as_strided(ops.fp4_cache_shape(pages, page, kv_heads, dim),
                                  (size + page_gap, size // page, size // page // kv_heads, 1))
            view.copy_(torch.from_numpy(raw).to(DEV).view(view.shape))
            self.caches.append(view)
        self.q = rng.standard_normal((len(lens) * m, heads, dim))
        self.bt = torch.from_numpy(self.table).to(DEV)
        self.sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.scale = dim ** -0.5

    def keys(self, b):
        n = self.lens[b]
        ids = self.table[b, :max(0, -(-n // self.page))]
        return [ref.unpack(raw[ids], self.Hkv, self.D, self.page, x == 1).reshape(-1, self.Hkv, self.D)[:n] for x, raw in enumerate(self.raw)]

    def run(self, dtype, out_dtype=None, fill=7.0):
        q = torch.from_numpy(self.q).to(dtype)
        out = torch.full(q.shape, fill, dtype=out_dtype or dtype, device=DEV)
        ws = ops.decode_fp4_workspace(len(self.lens), self.m, self.H, self.Hkv, self.D, DEV)
        ws[0].fill_(float("nan"))
        ws[1].fill_(float("nan"))
        ops.decode_attention_fp4(q.to(DEV), *self.caches, out, self.bt, self.sl, self.scale, ws, rows_per_request=self.m)
        return q, out

    def check(self, dtype, out_dtype=None):
        q, out = self.run(dtype, out_dtype)
        got, qd = out.double().cpu().numpy(), q.double().numpy()
        for b, n in enumerate(self.lens):
            rows = slice(b * self.m, (b + 1) * self.m)
            if n <= 0:
                assert (got[rows] == 7).all()
                continue
            o, av, ds = ref.attention(qd[rows], *self.keys(b), self.scale, self.m)
            there = np.arange(self.m) >= self.m - n
            assert (got[rows][~there] == 7).all()
            lim = ref.bound(o, av, ds, n, HALF[out_dtype or dtype])[there]
            err = np.abs(got[rows][there] - o[there])
            worst = float((err / lim).max())
            assert worst <= 1, (b, n, worst)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_decode_lengths(dtype, dim, page):
    """Lengths around every boundary: one key, a 16-key half, a tile, a page, pieces that split."""
    Batch(dim + page, [1, 2, 15, 16, 17, 31, 32, 33, 0, 63, 64, 65, 127, 129, 300, 1025, -3], 8, 2, dim, page).check(dtype)


@gpu
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (3, 1), (4, 4), (8, 1), (14, 2), (16, 1), (32, 8), (40, 2), (64, 1), (48, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_head_layouts(heads, kv_heads, dtype):
    Batch(heads * 10 + kv_heads, [700, 33, 0, 260], heads, kv_heads, 128, 16).check(dtype)
    Batch(heads * 10 + kv_heads, [41, 514], heads, kv_heads, 64, 32).check(dtype, torch.float32)


@gpu
@pytest.mark.parametrize("m", [2, 3, 4, 8, 16])
@pytest.mark.parametrize("dtype, dim", [(torch.bfloat16, 128), (torch.float16, 128), (torch.bfloat16, 64), (torch.float16, 64)])
def test_several_rows_per_request(m, dtype, dim):
    """Lengths below, at and above the number of rows; rows before the sequence's start are left alone."""
    Batch(m, [m - 1, m, m + 1, 1, 0, 32, 33, 47, 64 + m, 500], 8, 2, dim, 16, m=m).check(dtype)


@gpu
@pytest.mark.parametrize("batch", [64, 65, 130])
def test_many_requests(batch):
    """More requests than lanes that count them; empty ones among them, one that is much longer than the others."""
    rng = np.random.default_rng(batch)
    lens = [int(n) for n in rng.integers(-2, 90, batch)]
    lens[1], lens[batch // 2], lens[-1] = 0, 2000, 33
    Batch(batch, lens, 4, 1, 64, 16, m=2).check(torch.bfloat16)
    Batch(batch + 1, [0] * (batch - 1) + [5], 4, 2, 128, 16).check(torch.float16)


@gpu
def test_more_requests_than_workgroups():
    """Several requests to a workgroup and to a lane of the plan, some that lie in two spans."""
    rng = np.random.default_rng(5)
    lens = [int(n) for n in rng.integers(0, 40, 1100)]
    lens[700] = 900
    Batch(1100, lens, 2, 1, 64, 16).check(torch.bfloat16)


@gpu
def test_one_work_area_serves_steps_of_other_sizes():
    """What an earlier call left in the work area -- partial results, where its pieces lay -- does not reach a later one."""
    steps = [Batch(31, [900, 1, 64, 0, 2000], 8, 2, 128, 16), Batch(32, [33], 8, 2, 128, 16), Batch(33, [5, 700, 300], 8, 2, 128, 16, m=2),
             Batch(34, [0, 1500, 0, 40, 8], 8, 2, 128, 16)]
    ws = max((ops.decode_fp4_workspace(len(b.lens), b.m, 8, 2, 128, DEV) for b in steps), key=lambda w: w[0].numel())
    for b in steps * 3:
        q, want = b.run(torch.bfloat16)
        out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
        ops.decode_attention_fp4(q.to(DEV), *b.caches, out, b.bt, b.sl, b.scale, ws, rows_per_request=b.m)
        assert torch.equal(out, want)


@gpu
def test_few_long_sequences_split_over_the_chip():
    Batch(5, [20011], 8, 1, 128, 16).check(torch.bfloat16, torch.float32)
    Batch(6, [9000, 1, 12345], 4, 1, 128, 64, m=2).check(torch.float16, torch.float32)


@gpu
def test_page_stride_and_query_strides():
    b = Batch(8, [100, 45], 8, 2, 128, 16, page_gap=48)
    b.check(torch.bfloat16)
    # queries out of a fused projection, outputs into a wider row
    q = torch.from_numpy(b.q).to(torch.bfloat16)
    wide = torch.zeros(2, 20, 128, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:11] = q.to(DEV)
    out = torch.full((2, 12, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    ws = ops.decode_fp4_workspace(2, 1, 8, 2, 128, DEV)
    ops.decode_attention_fp4(wide[:, 3:11], *b.caches, out[:, 2:10], b.bt, b.sl, b.scale, ws)
    _, want = b.run(torch.bfloat16)
    assert torch.equal(out[:, 2:10], want) and (out[:, :2] == 7).all() and (out[:, 10:] == 7).all()


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_what_lies_behind_a_sequence_does_not_enter(dim):
    """Keys past the sequence -- stale tokens of its last page, other rows' pages -- hold NaN scales."""
    b = Batch(9, [37, 80], 8, 2, dim, 16)
    _, want = b.run(torch.bfloat16)
    for x, raw in enumerate(b.raw):
        nb = b.Hkv * b.page * dim // 2
        bad = raw.copy()
        bad[b.table[0, 2], nb:].reshape(b.Hkv, dim // 32, b.page)[:, :, 5:] = 255
        b.caches[x].copy_(torch.from_numpy(bad).to(DEV).view(b.caches[x].shape))
    _, got = b.run(torch.bfloat16)
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_nan_reaches_the_rows_that_see_it_and_no_other(dim, dtype):
    """Drafted rows: a NaN block in V (or K) of a later position must not reach earlier rows."""
    n, m, page = 45, 4, 16
    for in_v in (False, True):
        b = Batch(10, [n, 61], 8, 2, dim, page, m=m)
        _, want = b.run(dtype)
        nb = b.Hkv * page * dim // 2
        key, head, block = n - 2, 1, 1  # seen by rows 2 and 3
        raw = b.raw[in_v].copy()
        raw[b.table[0, key // page], nb:].reshape(b.Hkv, dim // 32, page)[head, block, key % page] = 255
        b.caches[in_v].copy_(torch.from_numpy(raw).to(DEV).view(b.caches[in_v].shape))
        _, got = b.run(dtype)
        nan = torch.isnan(got)
        hit = torch.zeros_like(nan)
        hit[2:4, 4:8, 32:64 if in_v else dim] = True
        if not in_v:
            hit[2:4, 4:8] = True
        assert torch.equal(nan, hit)
        assert torch.equal(got[~hit], want[~hit])


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(dim, dtype):
    for heads, m in ((8, 1), (8, 3), (32, 2)):
        b = Batch(16, [70, 33], heads, 2, dim, 16, m=m)
        _, want = b.run(dtype)
        b.q[0, 1, 5], b.q[1, heads - 1, dim - 1], b.q[m, 3, 0] = np.nan, np.inf, -np.inf
        _, got = b.run(dtype)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[0, 1], hit[1, heads - 1], hit[m, 3] = True, True, True
        assert torch.equal(torch.isnan(got), hit) and torch.equal(got[~hit], want[~hit])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_queries_and_keys_of_very_different_sizes(dtype):
    """Neighbouring query columns that differ by up to 2^19, keys scaled block by block: every product has to count in the
    scores as it does in an fp32 sum."""
    rng = np.random.default_rng(17)
    b = Batch(17, [300, 45, 1025], 8, 2, 128, 32, m=2)
    b.q *= np.ldexp(1.0, rng.integers(-13, 7, b.q.shape))
    for x in (0, 1):
        nb = b.Hkv * b.page * b.D // 2
        shift = rng.integers(-9, 5, b.raw[x][:, nb:].shape)
        b.raw[x][:, nb:] = np.clip(b.raw[x][:, nb:].astype(int) + shift, 1, 253).astype(np.uint8)
        b.caches[x].copy_(torch.from_numpy(b.raw[x]).to(DEV).view(b.caches[x].shape))
    b.scale = 0.01
    b.check(dtype, torch.float32)


@gpu
@pytest.mark.parametrize("seed", range(40))
def test_random_steps(seed):
    rng = np.random.default_rng(1000 + seed)
    kv = int(rng.choice([1, 2, 3, 4, 5, 8]))
    group = int(rng.integers(1, 17))
    m = int(rng.integers(1, max(2, min(9, 64 // group + 1))))
    batch = int(rng.choice([1, 2, 3, 7, 20]))
    lens = [int(n) for n in np.exp(rng.uniform(0, np.log(1500), batch)).astype(int)]
    if batch > 2:
        lens[int(rng.integers(batch))] = int(rng.integers(-1, 3))
    b = Batch(seed, lens, kv * group, kv, int(rng.choice([64, 128])), int(rng.choice([16, 32, 64, 256])), m=m,
              page_gap=int(rng.choice([0, 16, 80])))
    b.check([torch.bfloat16, torch.float16][seed % 2], [None, torch.float32][seed // 2 % 2])


@gpu
def test_pages_that_do_not_exist_count_as_nan():
    b = Batch(11, [40, 40, 90], 4, 1, 128, 16)
    _, want = b.run(torch.bfloat16)
    b.bt[0, 1] = 10 ** 6
    b.bt[2, 0] = -5
    q, got = b.run(torch.bfloat16)
    assert torch.isnan(got[0]).all() and torch.isnan(got[2]).all() and torch.equal(got[1], want[1])
    # a sequence longer than its row of the table
    b.bt.copy_(torch.from_numpy(b.table))
    out = torch.zeros_like(got)
    ops.decode_attention_fp4(q.to(DEV), *b.caches, out, b.bt[:, :3], b.sl, b.scale, ops.decode_fp4_workspace(3, 1, 4, 1, 128, DEV))
    assert torch.equal(out[:2], want[:2]) and torch.isnan(out[2]).all()
    k, v = ops.gather_dequant_kv_fp4(*b.caches, b.bt[:, :3], b.sl, torch.tensor([0, 40, 80], dtype=torch.int32, device=DEV), 170, 90, torch.bfloat16)
    assert torch.isnan(k[80 + 48:]).all() and torch.isnan(v[80 + 48:]).all() and not torch.isnan(k[:128]).any()


@gpu
@pytest.mark.parametrize("page", [16, 64])
def test_entries_past_a_sequence_are_not_used(page):
    """The table is looked up ahead of the tiles, past a sequence's last one too: what stands there does not matter, and a
    table just wide enough does as well."""
    lens = [32, 512, 1, 480, 33, 96]
    b = Batch(23, lens, 8, 2, 128, page)
    _, want = b.run(torch.bfloat16)
    width = max(-(-n // page) for n in lens)
    wide = torch.full((len(lens), width + 40), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
    for r, n in enumerate(lens):
        wide[r, :-(-n // page)] = b.bt[r, :-(-n // page)]
    for table in (wide, wide[:, :width], wide[:, :width].contiguous()):
        b.bt = table
        assert torch.equal(b.run(torch.bfloat16)[1], want)


@gpu
def test_a_table_without_columns():
    """Through the C interface (an empty tensor has no address): sequences with keys and no pages are NaN."""
    b = Batch(29, [3, 0, 40], 8, 2, 128, 16)
    q = torch.from_numpy(b.q).to(torch.bfloat16).to(DEV)
    out = torch.zeros_like(q)
    ws = ops.decode_fp4_workspace(3, 1, 8, 2, 128, DEV)
    a = _args(batch=3, q=q.data_ptr(), out=out.data_ptr(), k=b.caches[0].data_ptr(), v=b.caches[1].data_ptr(), max_blocks=0,
              block_table=b.bt.data_ptr(), seq_lens=b.sl.data_ptr(), partial_o=ws[0].data_ptr(), partial_ml=ws[1].data_ptr(),
              workspace_rows=ws[1].numel() // 2, num_pages=b.caches[0].shape[0], kv_stride_page=b.caches[0].stride(0))
    assert _lib.load().tmx_decode_attention_fp4(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == _lib.TMX_OK
    torch.cuda.synchronize()
    assert torch.isnan(out[0]).all() and torch.isnan(out[2]).all() and (out[1] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim, heads, page", [(128, 2, 16), (64, 3, 32), (128, 8, 64), (64, 1, 16)])
def test_gather_returns_the_values_the_cache_stands_for(dtype, dim, heads, page):
    lens = [1, 0, 16, 33, 130]
    b = Batch(12, lens, heads, heads, dim, page, page_gap=32)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    total = int(cu[-1])
    out = [torch.full((total + 3, heads, dim), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    got = ops.gather_dequant_kv_fp4(*b.caches, b.bt, b.sl, torch.from_numpy(cu).to(DEV), total, max(lens), dtype, out=out)
    for x in range(2):
        want = np.concatenate([b.keys(i)[x] for i in range(len(lens))])
        assert np.array_equal(got[x][:total].double().cpu().numpy(), want)  # exact: one fraction bit
        assert (got[x][total:] == 7).all()  # rows behind the last sequence
    # fewer rows than the sequences have: the rest is skipped
    out = [torch.full((total, heads, dim), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    ops.gather_dequant_kv_fp4(*b.caches, b.bt, b.sl, torch.from_numpy(cu).to(DEV), 50, max(lens), dtype, out=out)
    assert torch.equal(out[0][:50], got[0][:50]) and (out[0][50:] == 7).all()


@gpu
def test_caches_past_4_gib():
    """Pages half a GiB apart: every offset of the last ones needs more than 32 bits."""
    b = Batch(18, [100, 61], 8, 2, 128, 16, page_gap=(1 << 29) - 16 * 2 * 68)
    assert b.caches[0].stride(0) == 1 << 29 and int(b.table.max()) * (1 << 29) > 1 << 32
    b.check(torch.bfloat16)
    cu = torch.tensor([0, 100, 161], dtype=torch.int32, device=DEV)
    k, v = ops.gather_dequant_kv_fp4(*b.caches, b.bt, b.sl, cu, 161, 100, torch.bfloat16)
    for x, got in enumerate((k, v)):
        assert np.array_equal(got.double().cpu().numpy(), np.concatenate([b.keys(0)[x], b.keys(1)[x]]))
    rows = torch.randn(161, 2, 128, device=DEV).bfloat16()
    pos = [np.arange(n) for n in (100, 61)]
    slots = np.concatenate([b.table[i, p // 16].astype(np.int64) * 16 + p % 16 for i, p in enumerate(pos)])
    ops.reshape_and_cache_fp4(rows, -rows, *b.caches, torch.from_numpy(slots).to(DEV))
    k, v = ops.gather_dequant_kv_fp4(*b.caches, b.bt, b.sl, cu, 161, 100, torch.bfloat16)
    want = ref.values(*ref.quantise(rows.double().cpu().numpy()))
    assert np.array_equal(k.double().cpu().numpy(), want) and torch.equal(v, -k)
    # and the pages as pages
    last = int(b.table[:, :4].max())
    other = int((set(range(b.caches[0].shape[0])) - set(b.table.ravel().tolist())).pop())
    ops.copy_pages(b.caches, torch.tensor([[last, other]], device=DEV))
    assert torch.equal(b.caches[0][last], b.caches[0][other]) and torch.equal(b.caches[1][last], b.caches[1][other])


@gpu
def test_fp16_rows_saturate():
    x = torch.full((1, 1, 64), 65504.0, dtype=torch.float16, device=DEV)
    x[0, 0, 1] = -65504.0
    caches = [torch.zeros(ops.fp4_cache_shape(1, 16, 1, 64), dtype=torch.uint8, device=DEV) for _ in range(2)]
    ops.reshape_and_cache_fp4(x, x, *caches, torch.zeros(1, dtype=torch.int64, device=DEV))
    one, zero = torch.ones(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    k, v = ops.gather_dequant_kv_fp4(*caches, zero.view(1, 1), one, zero, 1, 1, torch.float16)
    assert torch.equal(k, x) and torch.equal(v, x)
    k, v = ops.gather_dequant_kv_fp4(*caches, zero.view(1, 1), one, zero, 1, 1, torch.bfloat16)
    assert k[0, 0, 0] == 65536 and v[0, 0, 1] == -65536


@gpu
def test_a_captured_step_replays_on_other_lengths():
    b = Batch(13, [700, 40, 1], 8, 2, 128, 16)
    q = torch.from_numpy(b.q).to(torch.bfloat16).to(DEV)
    out = torch.zeros_like(q)
    ws = ops.decode_fp4_workspace(3, 1, 8, 2, 128, DEV)
    key = torch.randn(3, 2, 128, device=DEV).bfloat16()
    slots = torch.full((3,), -1, dtype=torch.int64, device=DEV)

    def step():
        ops.reshape_and_cache_fp4(key, key, *b.caches, slots)
        ops.decode_attention_fp4(q, *b.caches, out, b.bt, b.sl, b.scale, ws)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for lens in ([700, 40, 1], [3, 0, 1], [650, 39, 1], [700, 40, 1]):
        b.sl.copy_(torch.tensor(lens, dtype=torch.int32))
        key.normal_()
        q.normal_()
        slots[0] = int(b.table[0, 0]) * 16 + 2
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.fill_(5.0)
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out), lens


@gpu
def test_runs_on_the_callers_stream():
    b = Batch(14, [900, 33], 8, 2, 128, 16)
    _, want = b.run(torch.bfloat16)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _, got = b.run(torch.bfloat16)
    s.synchronize()
    assert torch.equal(got, want)


@gpu
def test_refusals_on_the_gpu():
    b = Batch(15, [20], 8, 2, 128, 16)
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device=DEV)
    ws = ops.decode_fp4_workspace(1, 1, 8, 2, 128, DEV)

    def call(**kw):
        a = dict(q=q, k=b.caches[0], v=b.caches[1], out=torch.zeros_like(q), bt=b.bt, sl=b.sl, ws=ws, m=1)
        a.update(kw)
        return ops.decode_attention_fp4(a["q"], a["k"], a["v"], a["out"], a["bt"], a["sl"], 0.1, a["ws"], rows_per_request=a["m"])

    call()
    for bad in (dict(q=q.float(), out=q.float()), dict(out=q.half()), dict(q=q[..., :64], out=q[..., :64]), dict(sl=b.sl.long()),
                dict(bt=b.bt.long()), dict(bt=b.bt[0]), dict(ws=None), dict(ws=(ws[0][:8], ws[1])), dict(m=2), dict(m=0),
                dict(k=b.caches[0].to(torch.int8)), dict(k=b.caches[0][..., :34]), dict(q=q[:, :7], out=q[:, :7]),
                dict(k=b.caches[0].transpose(1, 2), v=b.caches[1].transpose(1, 2)), dict(sl=b.sl.cpu()), dict(ws=(ws[0].half(), ws[1]))):
        with pytest.raises(RuntimeError):
            call(**bad)
    rows = torch.zeros(2, 2, 128, dtype=torch.bfloat16, device=DEV)
    slots = torch.zeros(2, dtype=torch.int64, device=DEV)
    ops.reshape_and_cache_fp4(rows, rows, *b.caches, slots[:0])
    for bad in ((rows.float(), rows.float(), slots), (rows[:, :1], rows[:, :1], slots), (rows, rows[:1], slots), (rows, rows, slots.int()),
                (rows[..., :64], rows[..., :64], slots), (rows, rows.half(), slots), (rows, rows, slots.cpu())):
        with pytest.raises(RuntimeError):
            ops.reshape_and_cache_fp4(bad[0], bad[1], *b.caches, bad[2])
    cu = torch.tensor([0, 20], dtype=torch.int32, device=DEV)
    for bad in (dict(dt=torch.float32), dict(bt=b.bt.long()), dict(sl=b.sl.long()), dict(out=(rows, rows))):
        a = dict(dt=torch.bfloat16, bt=b.bt, sl=b.sl, out=None)
        a.update(bad)
        with pytest.raises(RuntimeError):
            ops.gather_dequant_kv_fp4(*b.caches, a["bt"], a["sl"], cu, 20, 20, a["dt"], out=a["out"])


# ------------------------------------------------------------------------------------------------ the backend
def test_backend_takes_the_mxfp4_cache_type():
    from vllm_trianglemix_amd.backend import TriangleMixAttentionBackend as B
    assert B.get_kv_cache_shape(11, 16, 8, 128, "mxfp4") == (2, 11, 16, 8, 68)
    assert B.get_kv_cache_shape(11, 16, 8, 128) == (2, 11, 16, 8, 128)
    impl = B.get_impl_cls()(32, 128, 0.1, 8, None, None, "mxfp4", None, "decoder", None, use_triangle=True)
    assert impl.fp4_cache and not impl.fp8_cache
    with pytest.raises(NotImplementedError):
        B.get_impl_cls()(32, 128, 0.1, 8, None, None, "int4", None, "decoder", None)


def _steps_metadata(builder, q_lens, seq_lens, table, slots, prompts=None):
    import types
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    m = types.SimpleNamespace(
        num_actual_tokens=int(cu[-1]), max_query_len=int(max(q_lens)), max_seq_len=int(max(seq_lens)),
        query_start_loc=torch.from_numpy(cu).to(DEV), query_start_loc_cpu=torch.from_numpy(cu),
        seq_lens=torch.tensor(seq_lens, dtype=torch.int32, device=DEV), seq_lens_cpu=torch.tensor(seq_lens, dtype=torch.int32),
        block_table_tensor=table, slot_mapping=slots)
    if prompts is not None:
        m.prompt_lens_cpu = np.asarray(prompts, np.int32)
    return builder.build(0, m)


def test_which_steps_the_backend_reads_in_place():
    import types
    from vllm_trianglemix_amd.backend import TriangleMixAttentionImpl, TriangleMixAttentionMetadata
    tri = TriangleMixAttentionImpl(32, 128, 0.1, 8, None, None, "mxfp4", None, "decoder", None, use_triangle=True)
    causal = TriangleMixAttentionImpl(32, 128, 0.1, 8, None, None, "mxfp4", None, "decoder", None, use_triangle=False)

    def md(q, s, uniform_decode=False, prompts=None):
        cu = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
        return TriangleMixAttentionMetadata(
            num_actual_tokens=int(cu[-1]), max_query_len=int(max(q)), query_start_loc=None, max_seq_len=int(max(s)), seq_lens=None,
            block_table=None, slot_mapping=None, query_start_loc_cpu=cu, seq_lens_cpu=np.asarray(s, np.int32), page_size=16,
            uniform_decode=uniform_decode, prompt_lens_cpu=None if prompts is None else np.asarray(prompts, np.int32))

    last = tri.pattern[2]
    for impl in (tri, causal):
        assert impl._fp4_rows_in_place(md([1, 1], [9, 5], True)) == 1
        assert impl._fp4_rows_in_place(md([4, 4], [9, 5])) == 4
        assert impl._fp4_rows_in_place(md([4, 3], [9, 5])) == 0
        assert impl._fp4_rows_in_place(md([17, 17], [90, 50])) == 0  # 68 rows per K/V head
    assert causal._fp4_rows_in_place(md([4, 4], [9, 5], prompts=[20, 5])) == 4
    assert tri._fp4_rows_in_place(md([4, 4], [9, 5], prompts=[20, 5])) == 0  # a chunk of a prompt, not its end
    narrow = TriangleMixAttentionImpl(32, 128, 0.1, 8, None, None, "mxfp4", None, "decoder", None, use_triangle=True, num_last_tokens=4)
    assert last > 4 and narrow._fp4_rows_in_place(md([4, 4], [9, 5])) == 0 and narrow._fp4_rows_in_place(md([3, 3], [9, 5])) == 3


@gpu
@pytest.mark.parametrize("dtype, D, H, Hkv", [(torch.bfloat16, 128, 8, 2), (torch.float16, 64, 4, 2)])
@pytest.mark.parametrize("use_triangle", [True, False])
def test_backend_serves_prompts_chunks_decode_and_drafts_from_a_4_bit_cache(dtype, D, H, Hkv, use_triangle):
    """Two prompts in one step, a third in two chunks, decode steps and a step of drafted rows out of one cache: every step against the formula over what the cache holds."""
    import types
    from oracle import trianglemix_oracle as orc
    from parity_tolerance import assert_close
    from vllm_trianglemix_amd.backend import TriangleMixAttentionBackend as B
    rng = np.random.default_rng(5)
    page, pages, gate = 16, 80, 64
    si, sl, last = 4, 32, 16
    impl = B.get_impl_cls()(H, D, D ** -0.5, Hkv, None, None, "mxfp4", None, "decoder", None, use_triangle=use_triangle,
                            num_sink_tokens=si, sliding_window_size=sl, num_last_tokens=last, short_sequence_gate=gate)
    builder = B.get_builder_cls()(types.SimpleNamespace(block_size=page), ["l0"], None, torch.device(DEV))
    kv = torch.zeros(B.get_kv_cache_shape(pages, page, Hkv, D, "mxfp4"), dtype=torch.uint8, device=DEV)
    order = rng.permutation(pages)
    table = np.zeros((3, 24), np.int32)
    for r in range(3):
        table[r] = order[24 * r:24 * r + 24]
    table_dev = torch.from_numpy(table).to(DEV)
    lens, held = [0, 0, 0], [[np.zeros((0, Hkv, D)) for _ in range(2)] for _ in range(3)]

    def step(q_lens, prompts=None, rows=None):
        live = [r for r in range(3) if q_lens[r]]
        ql = [q_lens[r] for r in live]
        T = sum(ql)
        q, k, v = (torch.from_numpy(rng.standard_normal((T, n, D))).to(dtype) for n in (H, Hkv, Hkv))
        slots, at = [], 0
        for r in live:
            pos = np.arange(lens[r], lens[r] + q_lens[r])
            slots.append(table[r, pos // page].astype(np.int64) * page + pos % page)
            for x, new in enumerate((k, v)):
                held[r][x] = np.concatenate([held[r][x], ref.values(*ref.quantise(new[at:at + q_lens[r]].double().numpy()))])
            at += q_lens[r]
            lens[r] += q_lens[r]
        sls = [lens[r] for r in live]
        m = _steps_metadata(builder, ql, sls, table_dev[live].contiguous(), torch.from_numpy(np.concatenate(slots)).to(DEV),
                            None if prompts is None else [prompts[r] for r in live])
        if rows is not None:
            assert impl._fp4_rows_in_place(m) == rows
        out = torch.zeros(T, H * D, dtype=dtype, device=DEV)
        impl.forward(None, q.to(DEV).view(T, -1), k.to(DEV).view(T, -1), v.to(DEV).view(T, -1), kv, m, out)
        cu = np.concatenate([[0], np.cumsum(ql)]).astype(np.int32)
        got = out.view(T, H, D).double().cpu().numpy()
        for i, r in enumerate(live):
            n = sls[i]
            full = n if prompts is None else max(n, prompts[r])
            mode = "triangle" if use_triangle and full > gate else "causal"
            kw = dict(full_lens=[full]) if full != n else {}
            want = orc.varlen_gqa_attention(q[cu[i]:cu[i + 1]].double().numpy(), lambda b: held[r][0], lambda b: held[r][1],
                                            [0, ql[i]], [n], D ** -0.5, mode, si, sl, last, **kw)
            assert_close(got[cu[i]:cu[i + 1]], want, "backend forward, 4-bit cache", out16=True)

    step([150, 40, 0], rows=0)
    step([1, 1, 0], rows=1)
    step([0, 0, 96], prompts=[0, 0, 200], rows=0)
    step([0, 0, 104], prompts=[0, 0, 200])
    step([1, 1, 1], rows=1)
    step([4, 4, 4], rows=4)
    step([1, 30, 2], rows=0)


@gpu
def test_backend_copies_blocks_of_all_layers():
    from vllm_trianglemix_amd.backend import TriangleMixAttentionBackend as B
    layers = [torch.randint(0, 256, B.get_kv_cache_shape(9, 16, 2, 64, "mxfp4"), dtype=torch.uint8, device=DEV) for _ in range(3)]
    want = [x.clone() for x in layers]
    B.copy_blocks(layers, torch.tensor([[1, 4], [1, 5], [2, 0]]))
    for x, y in zip(layers, want):
        y[:, [4, 5, 0]] = y[:, [1, 1, 2]]
        assert torch.equal(x, y)
