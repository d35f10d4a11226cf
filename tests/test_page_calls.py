"""How the page operators' calls reach the library: as plain functions of the extension, or through the registry where
something is to see them; what they refuse."""
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from vllm_trianglemix_amd import _lib, ops, torch_ops

gpu = pytest.mark.gpu
DEV = "cuda:0"
NAMES = ["trianglemix_free_pages", "trianglemix_fork_pages", "trianglemix_copy_pages", "trianglemix_compact_pages"]


def inputs():
    caches = [(torch.arange(12 * 64, device=DEV) % 251 + i).to(torch.uint8).view(12, 64) for i in range(3)]
    table = torch.tensor([[9, 3, -1], [7, 9, 11]], dtype=torch.int32, device=DEV)
    return caches, table, torch.tensor([20, 41], dtype=torch.int32, device=DEV)


def all_four(caches, table, lens):
    free, n = ops.free_pages(table, lens, 12, 16)
    child = ops.fork_pages(caches, table, lens, torch.tensor([1, 0], dtype=torch.int32, device=DEV), free[:2], 16)
    ops.copy_pages(caches, torch.tensor([[9, 5], [11, 6]], device=DEV))
    new, used = ops.compact_pages(caches, table, lens, 16)
    return [free, n, child, new, used, *caches]


def test_fake_tensors_never_reach_the_library():
    """They have no memory: nothing may take their address, whether a device is there or not.  The registry answers for them:
    a call without results is traced, the others say that they have no fake form."""
    with FakeTensorMode(), warnings.catch_warnings():
        warnings.simplefilter("error")
        caches, table, lens = inputs()
        assert ops.copy_pages(caches, table[:, :2].long().contiguous()) is None
        for call in (lambda: ops.free_pages(table, lens, 12, 16), lambda: ops.fork_pages(caches, table, lens, lens, lens, 16),
                     lambda: ops.compact_pages(caches, table, lens, 16), lambda: ops.compact_pages(tuple(caches), table, lens, 16)):
            with pytest.raises(_lib.TmxError, match="trianglemix_(free|fork|compact)_pages"):
                call()


def test_the_number_of_arguments_is_checked():
    torch_ops.load()
    t = torch.zeros(1, 2, dtype=torch.int64)
    m = torch_ops.module
    for f, right in ((m.copy_pages, 2), (m.free_pages, 4), (m.compact_pages, 4), (m.fork_pages, 6)):
        for n in (0, right - 1, right + 1):
            with pytest.raises(RuntimeError, match=f"takes {right} arguments"):
                f(*[t] * n)


@pytest.mark.parametrize("error, comes_as", [
    (torch.OutOfMemoryError, torch.OutOfMemoryError), (torch.AcceleratorError, torch.AcceleratorError), (RuntimeError, _lib.TmxError),
    (NotImplementedError, _lib.TmxError), (TypeError, _lib.TmxError), (KeyboardInterrupt, KeyboardInterrupt)])
def test_which_errors_are_refusals(monkeypatch, error, comes_as):
    """Callers tell memory that has run out (which they may free and try again) from arguments that are refused."""
    def raises(*args):
        raise error("what happened")

    torch_ops.load()
    monkeypatch.setattr(ops, "_require_gpu", lambda t, name: None)
    monkeypatch.setattr(torch_ops, "module", type("Module", (), dict.fromkeys(("free_pages", "copy_pages", "fork_pages", "compact_pages"), staticmethod(raises))))
    t = torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: ops.free_pages(t, t, 8, 16), lambda: ops.copy_pages([t], t), lambda: ops.fork_pages([t], t, t, t, t, 16),
                 lambda: ops.compact_pages([t], t, t, 16)):
        with pytest.raises(comes_as) as e:
            call()
        assert type(e.value) is comes_as


@pytest.mark.parametrize("big", [(1 << 32) + 16, (1 << 31) + 16])
def test_the_ctypes_binding_refuses_numbers_past_32_bits(monkeypatch, big):
    """It would cut them down to others: a page size of 2^32 + 16 to 16."""
    monkeypatch.setattr(ops, "_BINDING", "ctypes")
    monkeypatch.setattr(ops, "_require_gpu", lambda t, name: None)
    t, c = torch.zeros(1, 2, dtype=torch.int32), [torch.zeros(4, 32, dtype=torch.uint8)]
    lens = t[0, :1]
    for call in (lambda: ops.free_pages(t, lens, 8, big), lambda: ops.free_pages(t, lens, big, 16), lambda: ops.fork_pages(c, t, lens, lens, lens, big),
                 lambda: ops.compact_pages(c, t, lens, big)):
        with pytest.raises(RuntimeError, match="page_size"):
            call()
    k = torch.zeros(ops.fp4_cache_shape(2, 16, 1, 64), dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="max_seq_len"):
        ops.gather_dequant_kv_fp4(k, k, t, lens, lens, 4, big, torch.bfloat16)


@gpu
def test_modes_and_profilers_see_the_calls():
    want = all_four(*inputs())
    seen = []

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.__name__)
            return func(*args, **(kwargs or {}))

    class Function(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(getattr(func, "__name__", ""))
            return func(*args, **(kwargs or {}))

    for mode in (Dispatch, Function):
        seen.clear()
        with mode():
            got = all_four(*inputs())
        assert [n.split(".")[0] for n in seen if "pages" in n] == NAMES
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        got = all_four(*inputs())
    names = [e.name for e in prof.events()]
    assert all(any(n.endswith(x) for n in names) for x in NAMES)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # and a subclass of Tensor
    class Mine(torch.Tensor):
        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            seen.append(getattr(func, "__name__", ""))
            return super().__torch_function__(func, types, args, kwargs or {})

    seen.clear()
    caches, table, lens = inputs()
    ops.copy_pages([caches[0].as_subclass(Mine), *caches[1:]], torch.tensor([[9, 5]], device=DEV))
    assert any(n.startswith("trianglemix_copy_pages") for n in seen) and torch.equal(caches[0][9], caches[0][5])


@gpu
def test_plain_calls_stay_plain():
    caches, table, lens = inputs()
    m = torch_ops.module
    assert m.free_pages(table, lens, 12, 16) is not NotImplemented
    with torch.inference_mode():
        assert m.copy_pages(caches, torch.tensor([[9, 5]], device=DEV)) is None
    with torch.no_grad():
        assert m.compact_pages(caches, table, lens, 16) is not NotImplemented


@gpu
def test_pages_held_by_no_sequence_are_kept_by_a_row_of_their_own():
    """The null page 0, two blocks of a prefix cache and a request outside the batch: a row each, of whole pages."""
    page, pages = 16, 40
    table = torch.full((6, 4), -1, dtype=torch.int32)
    table[0, 0] = 0
    table[1, :2] = torch.tensor([33, 12])
    table[2, :3] = torch.tensor([39, 5, 20])
    table[3, :3], table[4, :2] = torch.tensor([33, 38, 7]), torch.tensor([30, 31])  # two sequences, one that shares page 33
    table[5, :4] = torch.tensor([1, 2, 3, 4])  # ended
    lens = torch.tensor([page, 2 * page, 3 * page, 37, 17, 0], dtype=torch.int32)
    start = [torch.randint(0, 256, (pages, 64), dtype=torch.uint8) for _ in range(2)]
    caches = [x.to(DEV) for x in start]
    t, n = table.to(DEV), lens.to(DEV)
    held = {0, 33, 12, 39, 5, 20, 38, 7, 30, 31}
    free, count = ops.free_pages(t, n, pages, page)
    assert set(free[:int(count)].tolist()) == set(range(pages)) - held
    new, used = ops.compact_pages(caches, t, n, page)
    assert int(used) == len(held) and int(new[0, 0]) == 0 and new[5].tolist() == [-1] * 4
    for r in range(5):
        for c in range(-(-int(lens[r]) // page)):
            for x, y in zip(start, caches):
                assert torch.equal(y[int(new[r, c])].cpu(), x[int(table[r, c])])
    assert int(new[1, 0]) == int(new[3, 0])
