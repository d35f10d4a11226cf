"""The 4-bit cache behind the backend: which memory its steps keep."""
import gc
import types
import weakref

import numpy as np
import pytest
import torch

from vllm_trianglemix_amd import ops
from vllm_trianglemix_amd.backend import TriangleMixAttentionBackend as B

gpu = pytest.mark.gpu
DEV = "cuda:0"


def common(q_lens, seq_lens, table=None, slots=None, device="cpu", prompts=None):
    """What the runner hands to the builder for a step."""
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    m = types.SimpleNamespace(
        num_actual_tokens=int(cu[-1]), max_query_len=int(max(q_lens)), max_seq_len=int(max(seq_lens)),
        query_start_loc=torch.from_numpy(cu).to(device), query_start_loc_cpu=torch.from_numpy(cu),
        seq_lens=torch.tensor(seq_lens, dtype=torch.int32, device=device), seq_lens_cpu=torch.tensor(seq_lens, dtype=torch.int32),
        block_table_tensor=torch.zeros(len(q_lens), 1, dtype=torch.int32) if table is None else table,
        slot_mapping=torch.zeros(int(cu[-1]), dtype=torch.int64) if slots is None else slots)
    if prompts is not None:
        m.prompt_lens_cpu = np.asarray(prompts, np.int32)
    return m


def builder_for(device, **config):
    return B.get_builder_cls()(types.SimpleNamespace(block_size=16), ["l0"], types.SimpleNamespace(**config), torch.device(device))


def layer(H, D, Hkv, **kw):
    return B.get_impl_cls()(H, D, D ** -0.5, Hkv, None, None, "mxfp4", None, "decoder", None, **kw)


class Recorder:
    """Stands in for the operators: what the layers call, with which memory."""

    def __init__(self, monkeypatch):
        self.areas, self.calls = [], []
        monkeypatch.setattr(ops, "decode_fp4_workspace", self.area)
        monkeypatch.setattr(ops, "reshape_and_cache_fp4", lambda *a: self.calls.append(("write", *a)))
        monkeypatch.setattr(ops, "decode_attention_fp4", lambda *a, rows_per_request: self.calls.append(("in place", rows_per_request, *a)))

    def area(self, batch, rows, num_heads, num_kv_heads, head_dim, device):
        t = torch.empty(1), torch.empty(1)
        self.areas.append(weakref.ref(t[0]))
        return t

    def alive(self):
        gc.collect()
        return sum(r() is not None for r in self.areas)


def test_work_areas_of_served_steps_do_not_add_up(monkeypatch):
    rec, builder = Recorder(monkeypatch), builder_for("cpu")
    H, D, Hkv = 8, 64, 2
    layers = [layer(H, D, Hkv, use_triangle=False), layer(H, D, Hkv, use_triangle=True)]
    kv = torch.zeros(B.get_kv_cache_shape(4, 16, Hkv, D, "mxfp4"), dtype=torch.uint8)

    def step(m):
        T = m.num_actual_tokens
        q, k, v = (torch.zeros(T, n * D, dtype=torch.bfloat16) for n in (H, Hkv, Hkv))
        for impl in layers:
            impl.forward(None, q, k, v, kv, m, q)
        used = [c[9][0] for c in rec.calls if c[0] == "in place"]
        rec.calls.clear()
        assert len(used) == 2 and used[0] is used[1]  # the step's layers share it
        return weakref.ref(used[0])

    for batch in range(1, 33):
        for rows in (1, 2, 5):
            step(builder.build(0, common([rows] * batch, [40] * batch)))
    assert len(rec.areas) >= 1 and rec.alive() <= 1
    # a captured step's stays where it is
    kept = step(builder.build_for_cudagraph_capture(common([1] * 4, [40] * 4)))
    for batch in range(1, 9):
        step(builder.build(0, common([1] * batch, [40] * batch)))
    assert kept() is not None
    assert step(builder.build_for_cudagraph_capture(common([1] * 4, [40] * 4)))() is kept()


@gpu
def test_a_captured_step_keeps_its_work_area_beside_other_steps():
    """Replays between eager steps of other sizes whose memory comes and goes."""
    rng = np.random.default_rng(1)
    H, D, Hkv, page, pages, batch = 8, 128, 2, 16, 256, 4
    builder, impl = builder_for(DEV), layer(H, D, Hkv, use_triangle=False)
    kv = torch.zeros(B.get_kv_cache_shape(pages, page, Hkv, D, "mxfp4"), dtype=torch.uint8, device=DEV)
    rows = torch.from_numpy(rng.standard_normal((pages * page, Hkv, D))).to(torch.bfloat16).to(DEV)
    ops.reshape_and_cache_fp4(rows, -rows, kv[0], kv[1], torch.arange(pages * page, device=DEV))
    table = torch.from_numpy(rng.permutation(pages).astype(np.int32).reshape(batch, -1)).to(DEV)

    def inputs(T):
        return [torch.from_numpy(rng.standard_normal((T, n * D))).to(torch.bfloat16).to(DEV) for n in (H, Hkv, Hkv)]

    # the runner's persistent buffers; no slot is written
    c = common([1] * batch, [900] * batch, table, torch.full((batch,), -1, dtype=torch.int64, device=DEV), DEV)
    q, k, v = inputs(batch)
    out = torch.zeros_like(q)
    md = builder.build_for_cudagraph_capture(c)
    impl.forward(None, q, k, v, kv, md, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        impl.forward(None, q, k, v, kv, md, out)
    del md
    for i in range(4):
        for m in (1, 3, 2 + i):
            lens = [int(x) for x in rng.integers(m, 1000, 3)]
            a = inputs(3 * m)
            step = builder.build(0, common([m] * 3, lens, table[:3], torch.full((3 * m,), -1, dtype=torch.int64, device=DEV), DEV))
            impl.forward(None, *a, kv, step, torch.zeros_like(a[0]))
            del step
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        scratch = torch.full((1 << 22,), float("nan"), device=DEV)  # what was freed is written over
        c.seq_lens.copy_(torch.from_numpy(rng.integers(1, 1001, batch).astype(np.int32)))
        for x, y in zip((q, k, v), inputs(batch)):
            x.copy_(y)
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = torch.zeros_like(out)
        impl.forward(None, q, k, v, kv, builder.build(0, c), eager)
        assert torch.equal(got, eager) and bool(torch.isfinite(got.float()).all())
        del scratch
