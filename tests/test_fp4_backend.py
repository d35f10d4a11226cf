"""The 4-bit cache behind the backend: which memory its steps keep, and mixed steps (running requests beside prompts)."""
import gc
import types
import weakref

import numpy as np
import pytest
import torch

import fp4_reference as ref
from vllm_trianglemix_amd import backend as be
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

        monkeypatch.setattr(ops, "gather_dequant_kv_fp4", self.gather)
        monkeypatch.setattr(ops, "attention", lambda *a, **kw: self.calls.append(("over rows", *a)))
        monkeypatch.setattr(be.TriangleMixAttentionMetadata, "block_index", lambda m, *a, **kw: m)
        monkeypatch.setattr(be.TriangleMixAttentionMetadata, "workspace", lambda m, *a: None)

    def gather(self, k, v, table, lens, cu, total, longest, dtype):
        self.calls.append(("read back", table, lens, cu, total, longest))
        return torch.empty(0), torch.empty(0)

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


def mixed(rec, builder, impl, q_lens, seq_lens, prompts=None):
    """The calls of a step: (requests, rows of each) in place, (row offsets, lengths) of those over rows read back."""
    T = sum(q_lens)
    table = torch.arange(len(q_lens), dtype=torch.int32).view(-1, 1)
    m = builder.build(0, common(q_lens, seq_lens, table, torch.arange(T), prompts=prompts))
    H, D, Hkv = impl.num_heads, impl.head_size, impl.num_kv_heads
    q = torch.arange(T, dtype=torch.float32).view(-1, 1).expand(T, H * D).contiguous()
    k = torch.zeros(T, Hkv * D)
    out = -q
    kv = torch.zeros(B.get_kv_cache_shape(4, 16, Hkv, D, "mxfp4"), dtype=torch.uint8)
    rec.calls.clear()
    impl.forward(None, q, k, k, kv, m, out)
    calls = {c[0]: c[1:] for c in rec.calls}
    assert calls["write"][4].tolist() == list(range(T))
    place = back = None
    at = 0
    if "in place" in calls:
        rows, cq, _, _, cout, ctable, clens = calls["in place"][:7]
        n = cq.shape[0] // rows
        place = n, rows
        assert cq[:, 0, 0].tolist() == list(range(n * rows)) == [-x for x in cout[:, 0, 0].tolist()]
        assert ctable[:n, 0].tolist() == list(range(n)) and clens[:n].tolist() == seq_lens[:n]
        at = n
    if "read back" in calls:
        rtable, lens, cu, total, longest = calls["read back"]
        aq, _, _, aout, rest, acu, alens = calls["over rows"][:7]
        first = sum(q_lens[:at])
        back = (acu.tolist(), lens.tolist())
        assert rtable[:, 0].tolist() == list(range(at, len(q_lens)))
        assert lens.tolist() == alens.tolist() == seq_lens[at:] == rest.seq_lens_cpu.tolist()
        assert acu.tolist() == np.concatenate([[0], np.cumsum(q_lens[at:])]).tolist() == rest.query_start_loc_cpu.tolist()
        assert cu.tolist() == np.concatenate([[0], np.cumsum(seq_lens[at:])]).tolist() and total == sum(seq_lens[at:]) and longest >= max(seq_lens[at:])
        assert aq[:, 0, 0].tolist() == list(range(first, T)) == [-x for x in aout[:, 0, 0].tolist()]
        assert rest.slot_mapping.tolist() == list(range(first, T)) and rest.num_actual_tokens == T - first
        assert rest.max_query_len == max(q_lens[at:])
        assert (rest.prompt_lens_cpu is None) == (prompts is None)
        if prompts is not None:
            assert rest.prompt_lens_cpu.tolist() == prompts[at:] == rest.prompt_lens.tolist()
    assert at * (place or (0, 0))[1] + (0 if back is None else back[0][-1]) == T
    return place, back


def test_requests_beside_a_prompt_are_not_read_back(monkeypatch):
    """A step of running requests and a chunk of a prompt: the cached rows of the former stay in 4 bits."""
    rec, builder = Recorder(monkeypatch), builder_for("cpu")
    causal, tri = layer(8, 128, 2, use_triangle=False), layer(8, 128, 2, use_triangle=True, num_last_tokens=4)
    long = [60000, 30000, 40000]  # 133 MB as 16-bit rows of 2 heads
    for impl in (causal, tri):
        place, back = mixed(rec, builder, impl, [1, 1, 1, 300], long + [700])
        assert place == (3, 1) and back == ([0, 300], [700])
        place, back = mixed(rec, builder, impl, [3, 3, 3, 1, 300], long + [9, 700])
        assert place == (3, 3) and back == ([0, 1, 301], [9, 700])
        assert mixed(rec, builder, impl, [300, 1, 1, 1], [700] + long)[0] is None  # (no running request at the beginning)
        assert mixed(rec, builder, impl, [1, 1, 300], [500, 40, 700])[0] is None  # little to read back: one call
        assert mixed(rec, builder, impl, [17, 17, 300], long)[0] is None  # 68 rows per K/V head
    # a triangle layer: rows past the trailing dense ones, and prompts that are not complete
    assert mixed(rec, builder, tri, [4, 4, 300], long)[0] is None and mixed(rec, builder, causal, [4, 4, 300], long)[0] == (2, 4)
    assert mixed(rec, builder, tri, [1, 1, 1, 9], long + [30], [60000, 30000, 50000, 30])[0] == (2, 1)
    assert mixed(rec, builder, causal, [1, 1, 1, 9], long + [30], [60000, 30000, 50000, 30])[0] == (3, 1)
    assert mixed(rec, builder, tri, [1, 1, 9], long, [60001, 30000, 40000])[0] is None
    # the switch that keeps decode requests on the block index keeps these too
    monkeypatch.setattr(be, "_DECODE_FIXED", False)
    assert mixed(rec, builder, causal, [1, 1, 1, 300], long + [700])[0] is None


def test_the_layers_of_a_mixed_step_share_its_second_part(monkeypatch):
    builder = builder_for("cpu")
    m = builder.build(0, common([1, 1, 30], [50, 60, 70]))
    assert m.after(2) is m.after(2) and m.after(1) is not m.after(2)
    assert m.leading_requests(1) == (2, 1) and m.leading_requests(0) == (0, 0)
    padded = builder.build(0, common([1, 1, 30], [50, 60, 70]))
    padded.num_actual_tokens = 40
    assert padded.leading_requests(4) == (0, 0)


def test_the_runner_is_asked_for_decode_requests_first():
    mx = builder_for("cpu", cache_config=types.SimpleNamespace(cache_dtype="mxfp4"))
    assert mx.reorder_batch_threshold == 1
    assert builder_for("cpu", cache_config=types.SimpleNamespace(cache_dtype="fp8")).reorder_batch_threshold is None
    assert builder_for("cpu").reorder_batch_threshold is None and B.get_builder_cls().reorder_batch_threshold is None


@pytest.mark.parametrize("D", [64, 128])
def test_a_cache_made_from_a_spec(D):
    """The way from a spec to the tensor that a runner takes (gpu_model_runner.py: bytes from the spec, blocks from the memory
    at hand, a raw tensor viewed as the backend's shape)."""
    spec = types.SimpleNamespace(block_size=32, num_kv_heads=8, head_size=D, dtype=torch.uint8,
                                 page_size_bytes=2 * 32 * 8 * (D // 2 + D // 32))
    raw = torch.zeros(11 * spec.page_size_bytes, dtype=torch.int8)
    assert raw.numel() % spec.page_size_bytes == 0
    shape = B.get_kv_cache_shape(raw.numel() // spec.page_size_bytes, spec.block_size, spec.num_kv_heads, spec.head_size, "mxfp4")
    cache = raw.view(spec.dtype).view(shape)
    k, v = cache.unbind(0)
    assert k.shape == ops.fp4_cache_shape(11, 32, 8, D) and k.stride(0) == v.stride(0) == spec.page_size_bytes // 2
    for bad in ((11, 32, 8, D // 2 + D // 32), (11, 48, 8, D)):
        with pytest.raises((RuntimeError, ValueError)):
            B.get_kv_cache_shape(*bad, "mxfp4")


def test_copies_without_layers_are_nothing():
    assert B.copy_blocks([], torch.tensor([[1, 2]])) is None


@gpu
@pytest.mark.parametrize("dtype, D, H, Hkv", [(torch.bfloat16, 128, 8, 2), (torch.float16, 64, 4, 2)])
@pytest.mark.parametrize("use_triangle", [True, False])
def test_mixed_steps_against_the_formula(monkeypatch, dtype, D, H, Hkv, use_triangle):
    from oracle import trianglemix_oracle as orc
    from parity_tolerance import assert_close
    monkeypatch.setattr(be, "_FP4_SPLIT_BYTES", 0)
    rng = np.random.default_rng(8)
    page, gate, si, sl, last = 16, 64, 4, 32, 16
    impl = layer(H, D, Hkv, use_triangle=use_triangle, num_sink_tokens=si, sliding_window_size=sl, num_last_tokens=last,
                 short_sequence_gate=gate)
    builder = builder_for(DEV)
    for q_lens, seq_lens, prompts, split in (
            ([1, 1, 40], [300, 17, 40], None, (2, 1)), ([1, 1, 1, 100, 3], [33, 500, 1, 180, 90], None, (3, 1)),
            ([3, 3, 70, 1], [200, 3, 150, 64], None, (2, 3)), ([1, 80, 1], [129, 200, 90], [100, 400, 90], (1, 1)),
            ([2, 2, 50], [120, 70, 90], [200, 70, 90], (0, 0) if use_triangle else (2, 2)), ([50, 1, 1], [60, 200, 300], None, (0, 0)),
            ([1, 1, 1, 17], [1, 2, 3, 17], None, (3, 1)), ([3, 3, 1, 1, 1], [80, 300, 65, 1, 400], None, (2, 3)),
            ([1] * 20 + [2, 2], list(range(3, 23)) + [200, 9], None, (20, 1))):
        T, R = sum(q_lens), len(q_lens)
        width = max(-(-n // page) for n in seq_lens)
        table = rng.permutation(R * width).astype(np.int32).reshape(R, width)
        held = [[rng.standard_normal((n, Hkv, D)) for _ in range(2)] for n in seq_lens]
        held = [[torch.from_numpy(x).to(dtype) for x in pair] for pair in held]
        kv = torch.zeros(B.get_kv_cache_shape(R * width, page, Hkv, D, "mxfp4"), dtype=torch.uint8, device=DEV)
        slots = [table[r, np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page for r, n in enumerate(seq_lens)]
        for r, (n, m) in enumerate(zip(seq_lens, q_lens)):
            if n > m:
                ops.reshape_and_cache_fp4(held[r][0][:n - m].to(DEV), held[r][1][:n - m].to(DEV), kv[0], kv[1], torch.from_numpy(slots[r][:n - m]).to(DEV))
        q = torch.from_numpy(rng.standard_normal((T, H, D))).to(dtype)
        new = [torch.cat([h[x][n - m:] for h, n, m in zip(held, seq_lens, q_lens)]).view(T, -1).to(DEV) for x in range(2)]
        c = common(q_lens, seq_lens, torch.from_numpy(table).to(DEV),
                   torch.from_numpy(np.concatenate([s[n - m:] for s, n, m in zip(slots, seq_lens, q_lens)])).to(DEV), DEV, prompts)
        md = builder.build(0, c)
        assert impl._fp4_leading_requests(md) == split
        out = torch.zeros(T, H * D, dtype=dtype, device=DEV)
        impl.forward(None, q.to(DEV).view(T, -1), *new, kv, md, out)
        got, at = out.view(T, H, D).double().cpu().numpy(), 0
        for r, (n, m) in enumerate(zip(seq_lens, q_lens)):
            full = n if prompts is None else max(n, prompts[r])
            kd, vd = (ref.values(*ref.quantise(x.double().numpy())) for x in held[r])
            kw = dict(full_lens=[full]) if full != n else {}
            want = orc.varlen_gqa_attention(q[at:at + m].double().numpy(), lambda b: kd, lambda b: vd, [0, m], [n], D ** -0.5,
                                            "triangle" if use_triangle and full > gate else "causal", si, sl, last, **kw)
            assert_close(got[at:at + m], want, "backend forward, 4-bit cache, mixed steps", out16=True)
            at += m


@gpu
def test_memory_of_a_mixed_step():
    """32 requests of 2000 cached tokens beside a short prompt: nothing of the size of their 16-bit rows is allocated."""
    H, D, Hkv, page, n, R = 8, 128, 2, 16, 2000, 32
    builder, impl = builder_for(DEV), layer(H, D, Hkv, use_triangle=False)
    width = n // page
    kv = torch.zeros(B.get_kv_cache_shape((R + 1) * width, page, Hkv, D, "mxfp4"), dtype=torch.uint8, device=DEV)
    table = torch.arange((R + 1) * width, dtype=torch.int32, device=DEV).view(R + 1, width)
    T = R + 40
    c = common([1] * R + [40], [n] * R + [40], table, torch.full((T,), -1, dtype=torch.int64, device=DEV), DEV)
    q, k = torch.zeros(T, H * D, dtype=torch.bfloat16, device=DEV), torch.zeros(T, Hkv * D, dtype=torch.bfloat16, device=DEV)
    out = torch.zeros_like(q)
    impl.forward(None, q, k, k, kv, builder.build(0, c), out)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    impl.forward(None, q, k, k, kv, builder.build(0, c), out)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 4 * R * n * Hkv * D // 4


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
