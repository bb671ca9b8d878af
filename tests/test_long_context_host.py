"""Long-context operators, what the host decides: frequencies, workspace sizes, refusals.  No GPU calls."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def built():
    import importlib
    import __graft_entry__ as entry
    entry.build()
    return importlib.import_module("mineru-diffusion_b200")


def freq(built, *args, **kw):
    f, factor = built.ops.rope_frequencies(*args, device="cpu", **kw)
    assert f.dtype == torch.float64
    return f, factor


def test_frequencies(built):
    plain, factor = freq(built, 128, 10000.0)
    assert factor == 1.0 and plain.shape == (64,)
    assert torch.allclose(plain, 10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128), rtol=1e-15)
    linear, _ = freq(built, 128, 10000.0, scaling={"type": "linear", "factor": 4})
    assert torch.equal(linear, plain / 4)
    # the raised base keeps the fastest and divides the slowest by the factor
    ntk, _ = freq(built, 128, 10000.0, scaling={"type": "ntk", "factor": 4})
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(plain[-1]) / 4, rel_tol=1e-12)


def test_frequencies_by_parts(built):
    length, s = 4096, 8.0
    plain, _ = freq(built, 64, 10000.0)
    f, factor = freq(built, 64, 10000.0, scaling={"type": "yarn", "factor": s, "original_max_position": length})
    assert math.isclose(factor, 0.1 * math.log(s) + 1)
    turns = length * plain / (2 * math.pi)
    ratio = plain / f
    assert bool((ratio[turns > 64] == 1).all()) and torch.allclose(ratio[turns < 0.5], torch.tensor(s, dtype=torch.float64))
    assert bool((ratio.diff() >= -1e-12).all()) and float(ratio.min()) >= 1 and float(ratio.max()) <= s + 1e-12
    _, given = freq(built, 64, scaling={"type": "yarn", "factor": s, "original_max_position": length, "attention_factor": 1.5})
    assert given == 1.5


def test_frequencies_refused(built):
    for args, kw in (((0,), {}), ((7,), {}), ((64,), {"scaling": {"type": "dynamic", "factor": 2}}), ((64,), {"scaling": {"type": "linear", "factor": 0.5}}),
                     ((2,), {"scaling": {"type": "ntk", "factor": 2}}), ((64,), {"scaling": {"type": "linear", "factor": float("nan")}})):
        with pytest.raises(ValueError):
            freq(built, *args, **kw)


def test_c_entries_refuse_before_any_launch(built):
    lib, at = built._lib.lib(), 64

    def shared(**o):
        a = built._lib.AttnSharedArgs(prefix_pages=2, table_stride=4, table_pages=4, num_pages=10, bs=2, block=8, hq=4, hkv=2, softmax_scale=0.1,
                                      workspace_bytes=1 << 40)
        for n in ("q", "k_cache", "v_cache", "out", "prefix_table", "prefix_len", "block_table", "ctx_lens", "workspace"):
            setattr(a, n, at)
        for n, v in o.items():
            setattr(a, n, v)
        return lib.mdb_attn_block_shared(ctypes.byref(a), None)

    assert shared(bs=0) == 0 and lib.mdb_attn_block_shared(None, None) == -1
    for o, code in (({"q": None}, -1), ({"prefix_table": None}, -1), ({"prefix_len": None}, -1), ({"hq": 5}, -1), ({"table_stride": 3}, -1), ({"table_pages": 0}, -1),
                    ({"bs": -1}, -1), ({"k_cache": 72}, -2), ({"workspace": 72}, -2), ({"hq": 258}, -3), ({"softmax_scale": 0.0}, -3), ({"bs": 70000}, -3),
                    ({"softmax_scale": float("nan")}, -3), ({"workspace_bytes": 100}, -5), ({"workspace": None}, -5)):
        assert shared(**o) == code, o

    def weights(**o):
        a = built._lib.KeyWeightsArgs(cols=100, table_stride=4, table_pages=4, num_pages=10, bs=2, block=8, hq=4, hkv=2, softmax_scale=0.1, decay=1.0)
        for n in ("q", "k_cache", "lse", "out", "block_table", "ctx_lens"):
            setattr(a, n, at)
        for n, v in o.items():
            setattr(a, n, v)
        return lib.mdb_key_weights(ctypes.byref(a), None)

    assert weights(bs=0) == 0 and lib.mdb_key_weights(None, None) == -1
    for o, code in (({"lse": None}, -1), ({"out": None}, -1), ({"cols": 0}, -1), ({"hq": 3}, -1), ({"table_stride": 1}, -1), ({"q": 72}, -2), ({"hq": 258}, -3),
                    ({"softmax_scale": -1.0}, -3), ({"cols": 1 << 40}, -3)):
        assert weights(**o) == code, o

    def evict(**o):
        a = built._lib.KvEvictArgs(bs=1, kv_heads=2, row_bytes=256, budget=10, recent=2, num_pages=4, table_stride=2, table_pages=2, weight_cols=100)
        for n in ("k_cache", "v_cache", "weights", "seqlens", "seqlens_out", "block_table", "kept"):
            setattr(a, n, at)
        for n, v in o.items():
            setattr(a, n, v)
        return lib.mdb_kv_evict(ctypes.byref(a), None)

    assert evict(bs=0) == 0 and lib.mdb_kv_evict(None, None) == -1
    for o, code in (({"recent": 11}, -1), ({"recent": -1}, -1), ({"budget": 0}, -1), ({"kept": None}, -1), ({"weights": None}, -1), ({"out_table": at}, -1),
                    ({"bs": 2, "table_stride": 1}, -1), ({"row_bytes": 24}, -2), ({"v_cache": 72}, -2), ({"bs": 40000}, -3), ({"row_bytes": 8192}, -3)):
        assert evict(**o) == code, o

    def rotary(**o):
        a = built._lib.RotaryEmbedArgs(dtype=0, n=2, heads=2, kv_heads=1, dim=64, rot_dims=64, q_out_row=128, q_out_head=64, k_out_row=64, k_out_head=64)
        for n in ("q", "k", "positions", "inv_freq", "q_out", "k_out"):
            setattr(a, n, at)
        for n, v in o.items():
            setattr(a, n, v)
        return lib.mdb_rotary_embed(ctypes.byref(a), None)

    assert rotary(n=0) == 0 and lib.mdb_rotary_embed(None, None) == -1
    for o, code in (({"dtype": 2}, -1), ({"rot_dims": 66}, -1), ({"rot_dims": 3}, -1), ({"k": None}, -1), ({"k_out": None}, -1), ({"v": at}, -1), ({"inv_freq": None}, -1),
                    ({"slots": at}, -1), ({"slots": at, "k_cache": at}, -1), ({"slots": at, "k_cache": at, "num_slots": 5, "v": at}, -1), ({"dim": 2048}, -3),
                    ({"heads": 70000}, -3), ({"q_out_row": 0}, -1), ({"q_out_head": 0}, -1), ({"k_out_row": 0}, -1)):
        assert rotary(**o) == code, o


def test_rotary_outputs_that_lie_on_one_another(built):
    """Row and head strides against the places they name.  Key heads past the limit: the call ends in a refusal either way."""
    import random
    lib, at, r = built._lib.lib(), 64, random.Random(5)

    def refused(n, heads, dim, row, head, kv_heads=40000, k_row=40000 * 4096, k_head=4096):
        a = built._lib.RotaryEmbedArgs(dtype=1, n=n, heads=heads, kv_heads=kv_heads, dim=dim, q_out_row=row, q_out_head=head, k_out_row=k_row, k_out_head=k_head)
        for f in ("q", "k", "positions", "q_out", "k_out"):
            setattr(a, f, at)
        code = lib.mdb_rotary_embed(ctypes.byref(a), None)
        assert code in (-1, -3)
        return code == -1

    seen = set()
    for _ in range(4000):
        n, heads, dim = r.randint(1, 7), r.randint(1, 7), r.choice([1, 2, 3, 8])
        row, head = r.randint(-40, 40), r.randint(-40, 40)
        places = [row * i + head * j + c for i in range(n) for j in range(heads) for c in range(dim)]
        apart = len(set(places)) == len(places)
        assert refused(n, heads, dim, row, head) is not apart, (n, heads, dim, row, head)
        seen.add(apart)
    assert seen == {True, False}
    big = 2 ** 62
    assert not refused(100, 50, 64, big, 64) and not refused(2 ** 31 - 1, 65536, 1024, 65536 * 1024, 1024) and refused(2 ** 31 - 1, 65536, 1024, 1024, 1024)
    assert refused(4, 2, 64, 128, 64, k_row=4096 * 39999, k_head=4096) and refused(4, 2, 64, 128, 64, k_row=63, k_head=4096)


def test_eviction_with_wide_weights_refused(built):
    lib, at = built._lib.lib(), 64

    def wide(cols, **o):
        a = built._lib.KvEvictArgs(bs=1, kv_heads=2, row_bytes=256, budget=10, recent=2, num_pages=4, table_stride=2, table_pages=2, weight_cols=100)
        for n in ("k_cache", "v_cache", "weights", "weights_out", "seqlens", "seqlens_out", "block_table", "kept"):
            setattr(a, n, at)
        for n, v in o.items():
            setattr(a, n, v)
        return lib.mdb_kv_evict_wide(ctypes.byref(a), cols, None)

    assert wide(10, bs=0) == 0 and lib.mdb_kv_evict_wide(None, 10, None) == -1
    assert wide(9) == -1 and wide(0) == -1 and wide(100, row_bytes=24) == -2 and wide(0, weights_out=None, row_bytes=24) == -2


def test_eviction_to_weights_that_lie_on_one_another(built):
    lib, at = built._lib.lib(), 64

    def code(bs, row, head, cols):      # rows of 8192 bytes: refused either way
        a = built._lib.KvEvictArgs(bs=bs, kv_heads=3, row_bytes=8192, budget=10, recent=2, num_pages=4, table_stride=2, table_pages=2, weight_cols=100,
                                   weight_out_row=row, weight_out_head=head)
        for n in ("k_cache", "v_cache", "weights", "weights_out", "seqlens", "seqlens_out", "block_table", "kept"):
            setattr(a, n, at)
        return lib.mdb_kv_evict_wide(ctypes.byref(a), cols, None)

    for bs, row, head, cols in ((1, 0, 10, 10), (1, 0, 12, 12), (4, 30, 10, 10), (4, 10, 40, 10), (4, 37, 12, 11)):
        assert code(bs, row, head, cols) == -3
    for bs, row, head, cols in ((1, 0, 10, 11), (1, 0, 0, 10), (4, 30, 10, 11), (4, 29, 10, 10), (4, 10, 0, 10), (4, 0, 10, 10), (2, 5, 100, 10)):
        assert code(bs, row, head, cols) == -1


def test_argument_blocks_keep_their_size(built):
    """Callers built against an earlier header pass blocks of these sizes; what came later (mdb_kv_evict_wide) is an argument of its own."""
    sizes = {'RotaryEmbedArgs': 208, 'AttnSharedArgs': 128, 'KeyWeightsArgs': 104, 'KvEvictArgs': 152}
    for name, size in sizes.items():
        assert ctypes.sizeof(getattr(built._lib, name)) == size, name


def test_workspace_of_the_shared_prefix(built):
    need = built.ops.shared_prefix_workspace_bytes
    assert need(0, 32, 16, 8) == 0 and need(4, 32, 16, 5) == 0
    rows = 4 * 32 * 16
    assert need(4, 32, 16, 8) >= 2 * rows * 130 * 4
    assert need(8, 32, 16, 8) > need(4, 32, 16, 8)


def test_room_of_a_workspace(built):
    room = built.ops._room
    x = torch.empty(6, 8)
    assert room(None) == 0 and room(x) == 192 and room(x[2:]) == 128 and room(x[0:0]) == 0 and room(x[:, :1].contiguous()) == 24
    for bad in (x[:1].expand(100, 8), x[:, ::2], x.t(), torch.empty(1, dtype=torch.uint8).expand(1 << 30)):
        with pytest.raises(ValueError):
            room(bad)


def test_wrappers_refuse_cpu_tensors(built):
    x = torch.zeros(2, 1, 64)
    with pytest.raises(RuntimeError):
        built.ops.rotary_embed(x, None, torch.arange(2), torch.ones(32, dtype=torch.float64))
    c = torch.zeros(1, 256, 1, 128, dtype=torch.bfloat16)
    q, n, t = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        built.ops.block_attn_shared_prefix(q, c, c, None, None, n, t)
    with pytest.raises(RuntimeError):
        built.ops.key_weights(q, c, torch.zeros(1, 1, 1), n, t)
    with pytest.raises(RuntimeError):
        built.ops.evict_kvcache(c, c, torch.zeros(1, 1, 256), n, t, 10)
