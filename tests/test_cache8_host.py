"""The 8-bit cache's refusals and host-side records on a CPU: no kernel runs here.

Tensors are CPU tensors that report a CUDA device; the C entry points check their arguments before they
touch the driver, so their refusals are tested through the library itself.
"""
import ctypes as C
from types import SimpleNamespace
from unittest.mock import patch

import pytest
import torch

from kvsnap_b200 import _abi, cache8

DEVICE = SimpleNamespace(type="cuda", index=0)


class OnCuda:
    """A CPU tensor that reports a CUDA device."""
    device = DEVICE

    def __init__(self, tensor, device=DEVICE):
        self._tensor, self.device = tensor, device

    def __getattr__(self, name):
        return getattr(self._tensor, name)


def layer(blocks=4, block_size=16, heads=2, dim=64, dtype=torch.float8_e4m3fn):
    return OnCuda(torch.zeros((2, blocks, block_size, heads, dim), dtype=dtype))


def scale(blocks=4, heads=2):
    return OnCuda(torch.zeros((blocks, 2, heads)))


@pytest.fixture
def make():
    real = torch.zeros

    def build(codes=None, scales=None):
        with patch.object(torch, "zeros", lambda *a, device=None, **k: real(*a, **k)):
            return cache8.PagedCache8(codes or {"l": layer()}, scales or {"l": scale()})
    return build


def batch(seqs=2, width=3, **kwargs):
    return cache8.PagedBatch(OnCuda(torch.zeros((seqs, width), dtype=torch.int32)),
                             OnCuda(torch.zeros(seqs + 1, dtype=torch.int32)),
                             OnCuda(torch.zeros(seqs, dtype=torch.int32)), **kwargs)


def rows(n=3, heads=2, dim=64, dtype=torch.bfloat16):
    return OnCuda(torch.zeros((n, heads, dim), dtype=dtype))


def test_records_describe_the_cache(make):
    storage = torch.zeros((6, 16, 2, 128), dtype=torch.float8_e4m3fn)                # K and V side by side
    view = storage.unflatten(3, (2, 64)).permute(3, 0, 1, 2, 4)
    cache = make({"l": OnCuda(view)}, {"l": scale(6)})
    record = cache._records["l"]
    assert (record.side_pitch, record.block_pitch, record.token_pitch, record.head_pitch) == (64, 4096, 256, 128)
    assert (record.blocks, record.block_size, record.kv_heads, record.head_dim) == (6, 16, 2, 64)
    assert record.codes == storage.data_ptr()


@pytest.mark.parametrize("codes,scales,match", [
    ({}, {}, "empty"),
    ({"a": layer()}, {"b": scale()}, "same layers"),
    ({"a": OnCuda(torch.zeros((2, 4, 16, 2, 64), dtype=torch.float8_e4m3fn), SimpleNamespace(type="cpu", index=None))},
     {"a": scale()}, "CUDA device"),
    ({"a": layer(dtype=torch.float8_e5m2)}, {"a": scale()}, "float8_e4m3fn"),
    ({"a": layer(dim=96)}, {"a": scale()}, "head_dim"),
    ({"a": layer(dim=256)}, {"a": scale()}, "head_dim"),
    ({"a": layer(block_size=8)}, {"a": scale()}, "block_size"),
    ({"a": layer(blocks=0)}, {"a": scale(0)}, "codes are"),
    ({"a": layer()}, {"a": scale(5)}, "scales"),
    ({"a": layer()}, {"a": OnCuda(torch.zeros((4, 2, 2), dtype=torch.float16))}, "scales"),
    ({"a": layer()}, {"a": OnCuda(torch.zeros((4, 2, 2)).transpose(1, 2))}, "scales"),
    ({"a": layer(), "b": layer(heads=1)}, {"a": scale(), "b": scale(heads=1)}, "layer b"),
    ({"a": OnCuda(torch.zeros((2, 4, 16, 2, 128), dtype=torch.float8_e4m3fn)[..., ::2])}, {"a": scale()}, "contiguous head_dim"),
    ({"a": OnCuda(torch.zeros((2, 4, 16, 2, 72), dtype=torch.float8_e4m3fn)[..., :64])}, {"a": scale()}, "16-byte"),
    ({"a": OnCuda(torch.zeros((2, 4, 16, 2, 80), dtype=torch.float8_e4m3fn)[..., 8:72])}, {"a": scale()}, "16-byte"),
])
def test_caches_it_refuses(make, codes, scales, match):
    if not codes:
        with pytest.raises(ValueError, match=match):
            cache8.PagedCache8(codes, scales)
        return
    with pytest.raises(ValueError, match=match):
        make(codes, scales)


def test_batches_it_refuses():
    good = dict(table=torch.zeros((2, 3), dtype=torch.int32), start=torch.zeros(3, dtype=torch.int32),
                lengths=torch.zeros(2, dtype=torch.int32))

    def build(max_query=None, device=DEVICE, **changes):
        made = {name: OnCuda(t, device) for name, t in {**good, **changes}.items()}
        return cache8.PagedBatch(made["table"], made["start"], made["lengths"], max_query=max_query)
    build()
    build(max_query=0)
    for changes in ({"table": good["table"].long()}, {"start": good["start"].long()}, {"lengths": good["lengths"].long()},
                    {"lengths": torch.zeros((2, 1), dtype=torch.int32)}, {"start": torch.zeros(2, dtype=torch.int32)},
                    {"table": torch.zeros((3, 3), dtype=torch.int32)}, {"table": torch.zeros((3, 2), dtype=torch.int32).t()},
                    {"device": SimpleNamespace(type="cpu", index=None)}, {"max_query": -1}, {"max_query": 1.0},
                    {"lengths": torch.zeros(4, dtype=torch.int32)[::2]}):
        with pytest.raises(ValueError):
            build(**changes)


@pytest.mark.parametrize("change,match", [
    ({"key": rows(dtype=torch.float32)}, "bfloat16 or float16"),
    ({"key": rows(heads=3)}, "key must be"),
    ({"key": rows(dim=128)}, "key must be"),
    ({"value": rows(n=4)}, "same rows"),
    ({"value": rows(dtype=torch.float16)}, "same rows and type"),
    ({"key": OnCuda(torch.zeros((3, 2, 128), dtype=torch.bfloat16)[..., ::2])}, "contiguous"),
    ({"key": OnCuda(torch.zeros((3, 2, 68), dtype=torch.bfloat16)[..., :64])}, "aligned"),
    ({"key": OnCuda(torch.zeros((3, 2, 64), dtype=torch.bfloat16), SimpleNamespace(type="cuda", index=1))}, "must be on"),
    ({"query": rows(heads=4)}, "needs rotary"),
    ({"query": rows(n=2, heads=4), "rotary": OnCuda(torch.zeros((9, 32, 2)))}, "query"),
    ({"rotary": OnCuda(torch.zeros((9, 32, 2), dtype=torch.float64))}, "rotary"),
    ({"rotary": OnCuda(torch.zeros((9, 32)))}, "rotary"),
    ({"rotary": OnCuda(torch.zeros((9, 40, 2)))}, "rotary_dim"),
    ({"rotary": OnCuda(torch.zeros((9, 4, 2)))}, "rotary_dim"),
    ({"rotary": OnCuda(torch.zeros((0, 32, 2)))}, "position"),
])
def test_appends_it_refuses(make, change, match):
    arguments = {"key": rows(), "value": rows(), **change}
    with pytest.raises(ValueError, match=match):
        make().append("l", arguments.pop("key"), arguments.pop("value"), batch(), **arguments)


def test_a_bound_of_rows_beyond_32_bits():
    """The C record's fields have 32 bits: a bound above the call's rows says no more than they do."""
    assert [batch(max_query=q)._for(7).max_query for q in (None, 2, 7, 2 ** 32 + 1)] == [7, 2, 7, 7]
    with pytest.raises(ValueError, match="too large"):
        batch(seqs=1, width=1 << 30)


def test_layers_and_devices_it_refuses(make):
    cache = make()
    with pytest.raises(KeyError, match="nowhere"):
        cache.append("nowhere", rows(), rows(), batch())
    with pytest.raises(KeyError, match="nowhere"):
        cache.attend("nowhere", rows(), batch())
    other = batch()
    other.device = SimpleNamespace(type="cuda", index=1)
    with pytest.raises(ValueError, match="batch must be on"):
        cache.append("l", rows(), rows(), other)


@pytest.mark.parametrize("query,out,match", [
    (rows(heads=3), None, "multiple"),
    (rows(heads=0), None, "multiple"),
    (rows(dtype=torch.float32), None, "bfloat16 or float16"),
    (rows(heads=4), rows(heads=2), "out must be"),
    (rows(heads=4), rows(heads=4, dtype=torch.float16), "out must be"),
    (rows(heads=4), OnCuda(torch.zeros((3, 4, 128), dtype=torch.bfloat16)[..., :64]), "out must be"),
    (rows(heads=4), OnCuda(torch.zeros(3 * 4 * 64 + 8, dtype=torch.bfloat16)[4:4 + 768].view(3, 4, 64)), "aligned"),
])
def test_attentions_it_refuses(make, query, out, match):
    with pytest.raises(ValueError, match=match):
        make().attend("l", query, batch(), out=out)


@pytest.mark.parametrize("caches,match", [
    ({}, "empty"),
    ({"l": layer(dtype=torch.float32)}, "bfloat16 or float16"),
    ({"l": layer(dim=128, dtype=torch.bfloat16)}, "16-bit cache must be"),
    ({"l": OnCuda(torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16))}, "16-bit cache must be"),
    ({"l": OnCuda(torch.zeros((2, 4, 16, 2, 68), dtype=torch.bfloat16)[..., :64])}, "aligned"),
    ({"l": layer(dtype=torch.bfloat16), "m": layer(dtype=torch.float16)}, "one type"),
])
def test_conversions_it_refuses(make, caches, match):
    cache = make({"l": layer(), "m": layer()}, {"l": scale(), "m": scale()})
    with pytest.raises(ValueError, match=match):
        cache.converter(caches)
    with pytest.raises(KeyError):
        cache.converter({"n": layer(dtype=torch.bfloat16)})


def test_rotary_tables():
    table = cache8.rotary_table(100001, 32, 10000.0, device="cpu")
    assert table.shape == (100001, 16, 2) and table.dtype == torch.float32
    angle = 100000 * 10000.0 ** (-2 * 3 / 32)
    assert table[100000, 3].tolist() == torch.tensor([torch.tensor(angle).double().cos(), torch.tensor(angle, dtype=torch.float64).sin()]).tolist() \
        or abs(table[100000, 3, 1].item() - torch.tensor(angle, dtype=torch.float64).sin().item()) < 2.0 ** -24
    for dim in (0, 8, 24):
        with pytest.raises(ValueError):
            cache8.rotary_table(4, dim, device="cpu")


# ---- the C entry points ----------------------------------------------------------------------


def library():
    from kvsnap_b200.dataplane import _dp, _load
    return _dp(_load())


def c_cache(**changes):
    fields = dict(codes=1 << 20, scales=1 << 20, side_pitch=1 << 16, block_pitch=2048, token_pitch=128, head_pitch=64,
                  blocks=4, block_size=16, kv_heads=2, head_dim=64, device=0, reserved=0)
    return _abi.C8Cache(**{**fields, **changes})


def c_batch(**changes):
    return _abi.C8Batch(**{**dict(table=4096, start=4096, lengths=4096, table_pitch=3, width=3, seqs=2, rows=3,
                                  max_query=3), **changes})


def append(lib, cache, batch, type=0, key=4096, pitch=256, q_heads=0, query=None, rotary=None, rotary_dim=0):
    return lib.kvsnap_c8_append(cache, batch, type, key, pitch, 128, 4096, 256, 128, query, 256, 128, q_heads, None,
                                rotary, 9, rotary_dim, 0, 4096, 0)


@pytest.mark.parametrize("cache,batch,more,message", [
    (c_cache(codes=0), c_batch(), {}, "no storage"),
    (c_cache(head_dim=96), c_batch(), {}, "head_dim"),
    (c_cache(block_size=24), c_batch(), {}, "block_size"),
    (c_cache(kv_heads=0), c_batch(), {}, "empty"),
    (c_cache(token_pitch=8), c_batch(), {}, "aligned"),
    (c_cache(), c_batch(table=0), {}, "no tables"),
    (c_cache(), c_batch(seqs=-1), {}, "invalid batch"),
    (c_cache(), c_batch(width=(1 << 26) + 1), {}, "2^30 tokens"),
    (c_cache(), c_batch(), {"key": 4104}, "aligned"),
    (c_cache(), c_batch(), {"key": None}, "aligned"),
    (c_cache(), c_batch(), {"pitch": 24}, "aligned"),
    (c_cache(), c_batch(), {"query": 4096}, "query"),
    (c_cache(), c_batch(), {"rotary": 4096, "rotary_dim": 72}, "rotary_dim"),
    (c_cache(), c_batch(), {"rotary": 4096, "rotary_dim": 128}, "rotary_dim"),
    (c_cache(), c_batch(rows=(1 << 31) - 1, seqs=1 << 30), {}, "too many rows"),
    (c_cache(), c_batch(), {"type": 2}, "type"),
])
def test_the_library_refuses_before_it_touches_a_device(cache, batch, more, message):
    lib = library()
    assert append(lib, cache, batch, **more) == -1
    assert message in lib.kvsnap_cuda_error().decode()
    if not more and "rows" not in message:
        assert lib.kvsnap_c8_attend(cache, batch, 0, 4096, 512, 128, 4, 1.0, 4096, None, 0, 4096, 0) == -1
        assert message in lib.kvsnap_cuda_error().decode()


def test_the_library_refuses_attentions_and_conversions():
    lib = library()
    for heads, out, message in ((3, 4096, "multiple"), (0, 4096, "multiple"), (4, None, "output"), (4, 4104, "aligned")):
        assert lib.kvsnap_c8_attend(c_cache(), c_batch(), 0, 4096, 512, 128, heads, 1.0, out, None, 0, 4096, 0) == -1
        assert message in lib.kvsnap_cuda_error().decode()
    for size, heads, dim, n, type, message in ((16, 2, 96, 1, 0, "head_dim"), (8, 2, 64, 1, 0, "block_size"),
                                               (16, 2, 64, -1, 0, "invalid"), (16, 2, 64, 1 << 33, 0, "too many"),
                                               (16, 2, 64, 1, 5, "type")):
        assert lib.kvsnap_c8_compress(4096, 1, size, heads, dim, type, 4096, 4096, n, -1, 4096, 0, 0) == -1
        assert message in lib.kvsnap_cuda_error().decode()
        assert lib.kvsnap_c8_expand(4096, 1, size, heads, dim, type, 4096, 4096, n, 4096, 0, 0) == -1
        assert message in lib.kvsnap_cuda_error().decode()


def test_the_workspace_s_size_needs_a_place_and_bounded_work():
    lib = library()
    assert lib.kvsnap_c8_attend_workspace(c_cache(), c_batch(), 4, None) == -1
    assert "place" in lib.kvsnap_cuda_error().decode()
    size = C.c_size_t(7)
    assert lib.kvsnap_c8_attend_workspace(c_cache(), c_batch(rows=0), 4, size) == 0 and size.value == 0
    assert lib.kvsnap_c8_attend_workspace(c_cache(), c_batch(seqs=1 << 20, width=1 << 20), 4, size) == -1
    assert "too much work" in lib.kvsnap_cuda_error().decode()


def test_calls_of_nothing_need_no_device():
    lib = library()
    assert append(lib, c_cache(), c_batch(rows=0)) == 0 and append(lib, c_cache(), c_batch(seqs=0)) == 0
    assert lib.kvsnap_c8_attend(c_cache(), c_batch(rows=0), 0, None, 0, 0, 4, 1.0, None, None, 0, 4096, 0) == 0
    assert lib.kvsnap_c8_compress(None, 0, 16, 2, 64, 0, None, None, 0, -1, 4096, 0, 0) == 0


def test_structures_have_the_header_s_sizes():
    assert C.sizeof(_abi.C8Cache) == 72 and C.sizeof(_abi.C8Batch) == 48 and C.sizeof(_abi.C8Pair) == 96


# ---- registration with the data plane ----------------------------------------------------------


def test_the_data_plane_registers_codes_and_scales():
    from kvsnap_b200.dataplane import TorchBlockDataPlane
    codes = {f"layers.{i}": layer(blocks=5, heads=4, dim=128) for i in range(2)}
    scales = {name: OnCuda(torch.zeros((5, 2, 4))) for name in codes}

    class View(OnCuda):
        def view(self, *shape):
            return View(self._tensor.view(*shape))

        def __getitem__(self, i):
            return View(self._tensor[i])

        def permute(self, *dims):
            return View(self._tensor.permute(*dims))

    wrap = lambda tensors: {name: View(t._tensor) for name, t in tensors.items()}   # noqa: E731
    with patch("kvsnap_b200.dataplane.CudaPool"):
        plane = TorchBlockDataPlane(wrap(codes), 16, 1 << 20, scales=wrap(scales))
        assert [l["name"] for l in plane.layers] == ["layers.0.k", "layers.0.scale", "layers.0.v", "layers.1.k",
                                                     "layers.1.scale", "layers.1.v"]
        assert [l["bytes"] for l in plane.layers[:3]] == [16 * 4 * 128, 2 * 4 * 4, 16 * 4 * 128]
        assert plane.layers[1]["shape"] == [1, 1, 8]
        for bad in (torch.zeros((5, 4, 2)).transpose(1, 2), torch.zeros((5, 8)), torch.zeros((5, 3, 4))):
            with pytest.raises(ValueError, match="scales"):
                TorchBlockDataPlane(wrap(codes), 16, 1 << 20, scales={"layers.0": View(bad)})
        with pytest.raises(ValueError, match="collides"):
            TorchBlockDataPlane({"a": View(torch.zeros((2, 4, 16, 2, 64))), "a.scale": View(torch.zeros((4, 2, 16, 64)))},
                                16, 1 << 20, scales={"a": View(torch.zeros((4, 2, 2)))})
        from kvsnap_b200.reshard import Regrouper
        with pytest.raises(ValueError, match="regrouped"):
            Regrouper(plane, None, 0)
