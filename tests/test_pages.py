"""Page operators (free / fork / compact / copy) against plain restatements on the host, and a serving run of them with the
4-bit cache's write and attention: prompt, fork, different continuations, end of some, closed-up pool, more steps."""
import ctypes

import numpy as np
import pytest
import torch

import fp4_reference as ref
from vllm_trianglemix_amd import _lib, ops

gpu = pytest.mark.gpu
DEV = "cuda:0"


# ------------------------------------------------------------------------------------------------ plain forms
def live_entries(table, lens, page):
    return [list(table[r, :min(table.shape[1], max(0, -(-int(n) // page)))]) for r, n in enumerate(lens)]


def plain_free(table, lens, pages, page):
    used = {int(e) for row in live_entries(table, lens, page) for e in row if 0 <= e < pages}
    free = [p for p in range(pages) if p not in used]
    return np.array(free + [-1] * (pages - len(free)), np.int32), len(free)


def plain_compact(table, lens, pages, page):
    free, n = plain_free(table, lens, pages, page)
    used = sorted(set(range(pages)) - set(free[:n].tolist()))
    U = len(used)
    move = dict(zip([p for p in used if p >= U], [int(p) for p in free[:n] if p < U]))
    new = np.full_like(table, -1)
    for r, row in enumerate(live_entries(table, lens, page)):
        new[r, :len(row)] = [move.get(int(e), int(e)) for e in row]
    return new, U, move


def plain_fork(table, lens, parents, fresh, page):
    child = np.full((len(parents), table.shape[1]), -1, np.int32)
    copies = []
    for i, r in enumerate(parents):
        if not 0 <= r < len(lens) or lens[r] <= 0:
            continue
        full, part = divmod(int(lens[r]), page)
        child[i, :full] = table[r, :full]
        if part and full < table.shape[1]:
            child[i, full] = fresh[i]
            copies.append((int(table[r, full]), int(fresh[i])))
    return child, copies


def random_tables(rng, rows, cols, pages, page, share=0.3):
    """Lengths from none to full; distinct pages, some shared between rows."""
    lens = rng.integers(0, cols * page + 1, rows)
    lens[rng.random(rows) < 0.25] = 0
    lens[rng.random(rows) < 0.1] = -3
    order = list(rng.permutation(pages))
    table = np.full((rows, cols), -1, np.int32)
    for r in range(rows):
        for c in range(max(0, -(-int(lens[r]) // page))):
            if rng.random() < share and r:
                table[r, c] = table[rng.integers(0, r), c]
            elif order:
                table[r, c] = order.pop()
    return table, lens.astype(np.int32)


def t32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(DEV)


# ------------------------------------------------------------------------------------------------ without a GPU
def test_the_plain_forms_agree_with_each_other():
    rng = np.random.default_rng(0)
    for _ in range(50):
        table, lens = random_tables(rng, 5, 7, 40, 4)
        new, U, move = plain_compact(table, lens, 40, 4)
        ids = {int(e) for row in live_entries(new, lens, 4) for e in row if e >= 0}
        assert ids == set(range(U)) and len(move) <= 20
        free, n = plain_free(new, lens, 40, 4)
        assert free[:n].tolist() == list(range(U, 40))


@pytest.mark.parametrize("change, code", [
    (dict(page_size=24), _lib.TMX_ERR_UNSUPPORTED), (dict(page_size=0), _lib.TMX_ERR_UNSUPPORTED), (dict(rows=-1), _lib.TMX_ERR_INVALID_ARG),
    (dict(num_pages=-1), _lib.TMX_ERR_INVALID_ARG), (dict(num_pages=1 << 31), _lib.TMX_ERR_UNSUPPORTED), (dict(table=None), _lib.TMX_ERR_INVALID_ARG),
    (dict(out=None), _lib.TMX_ERR_INVALID_ARG), (dict(rows=1 << 20, cols=1 << 20), _lib.TMX_ERR_UNSUPPORTED),
    (dict(rows=1 << 12, cols=1 << 10), _lib.TMX_ERR_INVALID_ARG),  # a large table without its work area
])
def test_plans_refuse_bad_arguments(change, code):
    c = dict(table=4096, rows=2, cols=4, page_size=16, num_pages=9, out=4096)
    c.update(change)
    lib = _lib.load()
    assert lib.tmx_free_pages(c["table"], c["cols"], c["rows"], c["cols"], c["table"], c["page_size"], c["num_pages"], c["out"], c["out"],
                              None, 0, None) == code
    assert lib.tmx_plan_compaction(c["table"], c["cols"], c["rows"], c["cols"], c["table"], c["page_size"], c["num_pages"], c["out"],
                                   c["out"], c["out"], None, 0, None) == code


@pytest.mark.parametrize("change, code", [
    (dict(size=24), _lib.TMX_ERR_UNSUPPORTED), (dict(stride=40), _lib.TMX_ERR_UNSUPPORTED), (dict(stride=16, size=32), _lib.TMX_ERR_INVALID_ARG),
    (dict(at=4104), _lib.TMX_ERR_INVALID_ARG), (dict(at=0), _lib.TMX_ERR_INVALID_ARG), (dict(size=0), _lib.TMX_ERR_INVALID_ARG),
    (dict(n=-1), _lib.TMX_ERR_INVALID_ARG), (dict(pairs=None), _lib.TMX_ERR_INVALID_ARG), (dict(n=2 ** 31 - 1, size=1 << 20, stride=1 << 20), _lib.TMX_ERR_UNSUPPORTED),
])
def test_copies_refuse_bad_arguments(change, code):
    c = dict(size=32, stride=32, at=4096, n=3, pairs=4096)
    c.update(change)
    at = (ctypes.c_void_p * 2)(c["at"], 4096)
    lib = _lib.load()
    assert lib.tmx_copy_pages(at, 2, c["size"], c["stride"], 9, c["pairs"], 32, c["n"], None, None) == code
    assert lib.tmx_fork_pages(at, 2, c["size"], c["stride"], 9, 4096, 4, 2, 4, 4096, 16, c["pairs"], c["pairs"], c["n"], 4096, None) == code


def test_empty_copies_are_nothing():
    lib = _lib.load()
    at = (ctypes.c_void_p * 1)(4096)
    assert lib.tmx_copy_pages(at, 1, 32, 32, 9, None, 32, 0, None, None) == 0
    assert lib.tmx_copy_pages(at, 1, 32, 32, 9, 4096, 16, 3, None, None) == _lib.TMX_ERR_UNSUPPORTED
    assert lib.tmx_fork_pages(at, 1, 32, 32, 9, 4096, 4, 2, 4, 4096, 16, None, None, 0, None, None) == 0
    assert lib.tmx_pages_work_ints(4, 4, 100) == 0 and lib.tmx_pages_work_ints(4096, 1024, 100) >= 10


def test_tensors_on_the_cpu_are_refused():
    bt, sl = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    c = [torch.zeros(8, 64, dtype=torch.uint8)]
    for call in (lambda: ops.free_pages(bt, sl, 8, 16), lambda: ops.copy_pages(c, torch.zeros(1, 2, dtype=torch.int64)),
                 lambda: ops.fork_pages(c, bt, sl, sl, sl, 16), lambda: ops.compact_pages(c, bt, sl, 16)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


# ------------------------------------------------------------------------------------------------ on the GPU
# (rows, columns, pages, page size): one workgroup makes the plan of the first ones, launches over the chip that of the last
PLANS = [(1, 1, 1, 16), (3, 5, 31, 16), (4, 9, 32, 1), (6, 8, 64, 16), (5, 40, 161, 4), (40, 33, 2000, 16), (1500, 50, 70001, 16), (2, 40000, 70016, 16)]


@gpu
@pytest.mark.parametrize("rows, cols, pages, page", PLANS)
def test_free_pages(rows, cols, pages, page):
    rng = np.random.default_rng(rows * cols)
    for k in range(3):
        table, lens = random_tables(rng, rows, cols, pages, page)
        if k == 1:
            lens[:] = 0  # nothing runs
        if k == 2:  # entries that are no pages
            table[rng.random(table.shape) < 0.1] = pages + 5
            table[rng.random(table.shape) < 0.1] = -7
        free, n = ops.free_pages(t32(table), t32(lens), pages, page)
        want, count = plain_free(table, lens, pages, page)
        assert int(n) == count and np.array_equal(free.cpu().numpy(), want)


@gpu
@pytest.mark.parametrize("rows, cols, pages, page", PLANS)
@pytest.mark.parametrize("caches", [1, 5])
def test_compact_pages(rows, cols, pages, page, caches):
    rng = np.random.default_rng(rows * cols + caches)
    for k in range(3):
        table, lens = random_tables(rng, rows, cols, pages, page)
        if k == 1:
            lens[:] = 0
        if k == 2:
            table[rng.random(table.shape) < 0.05] = pages
        start = [torch.randint(0, 256, (pages, 4, 12), dtype=torch.uint8) for _ in range(caches)]
        got = [x.to(DEV) for x in start]
        new, count = ops.compact_pages(got, t32(table), t32(lens), page)
        want, U, move = plain_compact(table, lens, pages, page)
        assert int(count) == U and np.array_equal(new.cpu().numpy(), want)
        for x, y in zip(start, got):
            if move:
                x[list(move.values())] = x[list(move.keys())]
            assert torch.equal(y.cpu(), x)


@gpu
@pytest.mark.parametrize("shape, dtype", [((16,), torch.uint8), ((16, 3, 68), torch.uint8), ((16, 2, 64), torch.bfloat16), ((7, 3, 16), torch.float32),
                                          ((33, 17, 16), torch.float16), ((64, 8, 128), torch.bfloat16)])
@pytest.mark.parametrize("bits", [torch.int32, torch.int64])
def test_copy_pages(shape, dtype, bits):
    """Pages of odd numbers of 16-byte units, of one and of several chunks; views with a page stride of their own."""
    rng = np.random.default_rng(len(shape))
    pages = 23
    whole = torch.randint(-1000, 1000, (3, pages, 2, *shape)).to(dtype).to(DEV)
    views = [whole[i, :, j] for i in range(3) for j in range(2)]  # K and V of a layer side by side, page by page
    start = whole.clone()
    perm = rng.permutation(pages)
    src, dst = perm[:5].repeat(2), perm[5:15]
    pairs = np.stack([src, dst], 1).tolist() + [[-1, 3], [int(perm[20]), pages], [4, -2], [10 ** 6, 1]]
    ops.copy_pages(views, torch.tensor(pairs, dtype=bits, device=DEV))
    start[:, torch.from_numpy(dst)] = start[:, torch.from_numpy(src)]
    assert torch.equal(whole, start)
    ops.copy_pages(views, torch.zeros(0, 2, dtype=bits, device=DEV))
    ops.copy_pages([], torch.zeros(1, 2, dtype=bits, device=DEV))
    assert torch.equal(whole, start)


@gpu
def test_more_caches_than_one_launch_takes():
    whole = torch.randint(0, 256, (300, 6, 48), dtype=torch.uint8, device=DEV)
    start = whole.clone()
    ops.copy_pages(list(whole), torch.tensor([[0, 3], [1, 5]], device=DEV))
    start[:, [3, 5]] = start[:, [0, 1]]
    assert torch.equal(whole, start)
    bt, sl = t32([[0, 1], [2, -1]]), t32([20, 5])
    child = ops.fork_pages(list(whole), bt, sl, t32([0, 1, 0]), t32([3, 4, 5]), 16)
    start[:, [3, 4, 5]] = start[:, [1, 2, 1]]
    assert torch.equal(whole, start) and child.tolist() == [[0, 3], [4, -1], [0, 5]]


@gpu
@pytest.mark.parametrize("shape", [(3, 32), (16, 8, 68)])
@pytest.mark.parametrize("rows, cols, page, children", [(1, 1, 16, 1), (3, 5, 16, 7), (8, 300, 16, 40), (4, 9, 1, 5), (5, 6, 64, 3)])
def test_fork_pages(rows, cols, page, children, shape):
    rng = np.random.default_rng(rows + cols)
    pages = rows * cols + children + 3
    table, lens = random_tables(rng, rows, cols, pages - children, page, share=0.0)
    if rows > 2:
        lens[0], lens[1] = cols * page, (cols - 1) * page  # ends on a page boundary: nothing to copy
        table[0] = -1
        order = rng.permutation(pages - children)
        table[0], table[1, :cols - 1] = order[:cols], order[cols:2 * cols - 1] if 2 * cols - 1 <= len(order) else order[:cols - 1]
    parents = rng.integers(0, rows, children).astype(np.int32)
    if children > 3:
        parents[1], parents[2] = -1, rows  # no such row
    fresh = np.arange(pages - children, pages).astype(np.int32)
    start = [torch.randint(0, 256, (pages, *shape), dtype=torch.uint8) for _ in range(4)]
    got = [x.to(DEV) for x in start]
    child = ops.fork_pages(got, t32(table), t32(lens), t32(parents), t32(fresh), page)
    want, copies = plain_fork(table, lens, parents, fresh, page)
    assert np.array_equal(child.cpu().numpy(), want)
    for x, y in zip(start, got):
        for a, b in copies:
            if a >= 0:
                x[b] = x[a]
        assert torch.equal(y.cpu(), x)
    # without caches: the tables alone
    assert np.array_equal(ops.fork_pages([], t32(table), t32(lens), t32(parents), t32(fresh), page).cpu().numpy(), want)


@gpu
def test_captured_page_operators_replay_on_other_tables():
    rng = np.random.default_rng(3)
    caches = list(torch.randint(0, 256, (4, 64, 160), dtype=torch.uint8, device=DEV))
    bt, sl = torch.zeros(6, 9, dtype=torch.int32, device=DEV), torch.zeros(6, dtype=torch.int32, device=DEV)
    parents = t32([0, 1])
    ops.compact_pages(caches, bt, sl, 16)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        free, n = ops.free_pages(bt, sl, 64, 16)
        child = ops.fork_pages(caches, bt, sl, parents, free[:2], 16)
        new, U = ops.compact_pages(caches, bt, sl, 16)
    for _ in range(4):
        table, lens = random_tables(rng, 6, 9, 60, 16)
        bt.copy_(t32(table))
        sl.copy_(t32(lens))
        before = [c.cpu() for c in caches]
        g.replay()
        torch.cuda.synchronize()
        wf, wn = plain_free(table, lens, 64, 16)
        wc, copies = plain_fork(table, lens, [0, 1], wf[:2], 16)
        wt, wu, move = plain_compact(table, lens, 64, 16)
        assert np.array_equal(free.cpu().numpy(), wf) and int(n) == wn and np.array_equal(child.cpu().numpy(), wc)
        assert np.array_equal(new.cpu().numpy(), wt) and int(U) == wu
        for x, y in zip(before, caches):
            for a, b in copies:
                if a >= 0:
                    x[b] = x[a]
            if move:
                x[list(move.values())] = x[list(move.keys())]
            assert torch.equal(y.cpu(), x)


@gpu
def test_empty_tables():
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    c = [torch.arange(5 * 32, dtype=torch.uint8, device=DEV).view(5, 32)]
    for bt in (torch.zeros(0, 4, dtype=torch.int32, device=DEV), torch.zeros(0, 0, dtype=torch.int32, device=DEV)):
        free, n = ops.free_pages(bt, none, 5, 16)
        assert free.tolist() == [0, 1, 2, 3, 4] and int(n) == 5
        table, used = ops.compact_pages(c, bt, none, 16)
        assert table.shape == bt.shape and int(used) == 0
        assert ops.fork_pages(c, bt, none, none, none, 16).shape == bt.shape
    free, n = ops.free_pages(torch.zeros(2, 4, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV), 0, 16)
    assert free.numel() == 0 and int(n) == 0
    assert torch.equal(c[0].flatten().cpu(), torch.arange(5 * 32, dtype=torch.uint8))


@gpu
def test_the_registered_operators_do_the_same():
    from vllm_trianglemix_amd import torch_ops
    C = torch_ops.load()
    rng = np.random.default_rng(6)
    table, lens = random_tables(rng, 6, 9, 60, 16)
    start = torch.randint(0, 256, (3, 64, 48), dtype=torch.uint8, device=DEV)
    bt, sl = t32(table), t32(lens)
    one, two = list(start.clone()), list(start.clone())
    free, n = ops.free_pages(bt, sl, 64, 16)
    free2, n2 = C.trianglemix_free_pages(bt, sl, 64, 16)
    assert torch.equal(free, free2) and int(n) == int(n2)
    parents = t32([0, 3])
    assert torch.equal(ops.fork_pages(one, bt, sl, parents, free[:2], 16), C.trianglemix_fork_pages(two, bt, sl, parents, free[:2], 16))
    a, b = ops.compact_pages(one, bt, sl, 16), C.trianglemix_compact_pages(two, bt, sl, 16)
    assert torch.equal(a[0], b[0]) and int(a[1]) == int(b[1])
    pairs = torch.tensor([[1, 60], [2, 61]], device=DEV)
    ops.copy_pages(one, pairs)
    C.trianglemix_copy_pages(two, pairs)
    assert torch.equal(torch.stack(one), torch.stack(two))
    with pytest.raises(RuntimeError):
        C.trianglemix_copy_pages(two, pairs.float())
    for bad in ((one, None), (pairs, pairs), ([pairs, 3], pairs), (one,)):
        with pytest.raises(RuntimeError):
            torch_ops.module.copy_pages(*bad)


@gpu
def test_refusals_on_the_gpu():
    bt, sl = torch.zeros(2, 4, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    c = [torch.zeros(8, 64, dtype=torch.uint8, device=DEV) for _ in range(2)]
    p = torch.zeros(1, 2, dtype=torch.int64, device=DEV)
    for call in (lambda: ops.free_pages(bt.long(), sl, 8, 16), lambda: ops.free_pages(bt, sl.long(), 8, 16), lambda: ops.free_pages(bt, sl, 8, 17),
                 lambda: ops.free_pages(bt, sl, -1, 16), lambda: ops.free_pages(bt[:1], sl, 8, 16), lambda: ops.free_pages(bt, sl.cpu(), 8, 16),
                 lambda: ops.copy_pages(c, p.float()), lambda: ops.copy_pages(c, p[0]), lambda: ops.copy_pages([c[0], c[1][:4]], p),
                 lambda: ops.copy_pages([c[0], c[1].cpu()], p), lambda: ops.copy_pages([c[0], c[1].float()], p),
                 lambda: ops.copy_pages([c[0][:, ::2]], p), lambda: ops.copy_pages([c[0][:, :24]], p), lambda: ops.copy_pages([c[0][:, 8:24]], p),
                 lambda: ops.compact_pages([], bt, sl, 16), lambda: ops.fork_pages(c, bt, sl, sl, sl[:1], 16),
                 lambda: ops.fork_pages(c, bt, sl, sl.long(), sl, 16), lambda: ops.fork_pages(c, bt, sl, sl, sl, 12)):
        with pytest.raises(RuntimeError):
            call()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_serving_run(dtype):
    """Two prompts; four samples forked from them; every sample decodes its own tokens; half of them end; the pool is
    closed up; the others go on, also with several rows a step.  All layers' caches are moved together, each step's
    attention is compared with the sequence's own keys kept on the host."""
    rng = np.random.default_rng(4)
    H, Hkv, D, page, pages, layers, cols = 8, 2, 128, 16, 40, 3, 12
    shape = ops.fp4_cache_shape(pages, page, Hkv, D)
    kc = [torch.zeros(shape, dtype=torch.uint8, device=DEV) for _ in range(layers)]
    vc = [torch.zeros(shape, dtype=torch.uint8, device=DEV) for _ in range(layers)]
    everything = kc + vc
    table = torch.full((0, cols), -1, dtype=torch.int32, device=DEV)
    lens = []
    kept = []  # per sequence, per layer: K and V values as the cache holds them

    def rows(n):
        return torch.from_numpy(rng.standard_normal((n, Hkv, D))).to(dtype)

    def write(seq, n):
        """n more tokens of a sequence, with pages for them"""
        nonlocal table
        have, need = -(-lens[seq] // page), -(-(lens[seq] + n) // page)
        if need > have:
            free, count = ops.free_pages(table, t32(lens), pages, page)
            assert int(count) >= need - have
            table[seq, have:need] = free[:need - have]
        pos = torch.arange(lens[seq], lens[seq] + n, device=DEV)
        slots = table[seq].long()[pos // page] * page + pos % page
        for x in range(layers):
            k, v = rows(n), rows(n)
            ops.reshape_and_cache_fp4(k.to(DEV), v.to(DEV), kc[x], vc[x], slots)
            for y, r in enumerate((k, v)):
                kept[seq][x][y] = np.concatenate([kept[seq][x][y], ref.values(*ref.quantise(r.double().numpy()))])
        lens[seq] += n

    def attend(m):
        live = [s for s in range(len(lens)) if lens[s]]
        q = torch.from_numpy(rng.standard_normal((len(live) * m, H, D))).to(dtype)
        for x in range(layers):
            out = torch.zeros(q.shape, dtype=torch.float32, device=DEV)
            ops.decode_attention_fp4(q.to(DEV), kc[x], vc[x], out, table[live].contiguous(), t32([lens[s] for s in live]), D ** -0.5,
                                     ops.decode_fp4_workspace(len(live), m, H, Hkv, D, DEV), rows_per_request=m)
            for i, s in enumerate(live):
                o, av, ds = ref.attention(q[i * m:(i + 1) * m].double().numpy(), *kept[s][x], D ** -0.5, m)
                assert (np.abs(out[i * m:(i + 1) * m].double().cpu().numpy() - o) <= ref.bound(o, av, ds, lens[s], 2.0 ** -24)).all(), (s, x)

    def start(row):
        nonlocal table
        table = torch.cat([table, row.view(1, cols)])
        lens.append(0)
        kept.append([[np.zeros((0, Hkv, D)) for _ in range(2)] for _ in range(layers)])

    for n in (37, 48):  # one ends inside a page, one on a boundary
        start(torch.full((cols,), -1, dtype=torch.int32, device=DEV))
        write(len(lens) - 1, n)
    attend(1)
    parents = [0, 0, 1, 0]
    free, _ = ops.free_pages(table, t32(lens), pages, page)
    child = ops.fork_pages(everything, table, t32(lens), t32(parents), free[:4].contiguous(), page)
    for i, p in enumerate(parents):
        start(child[i])
        lens[-1] = lens[p]
        kept[-1] = [[a.copy() for a in x] for x in kept[p]]
    attend(1)
    for step in range(3):
        for s in range(len(lens)):
            write(s, 1 + step)
        attend(1 + step)
    for s in (0, 3):
        lens[s] = 0  # ended: its pages are free, unless a sample still shares them
    table, count = ops.compact_pages(everything, table, t32(lens), page)
    assert int(table.max()) < int(count) == len({int(e) for s in range(len(lens)) for e in table[s, :-(-lens[s] // page)]})
    attend(2)
    for s in (1, 2, 4, 5):
        write(s, 9)
    attend(4)
