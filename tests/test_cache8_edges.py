"""What the 8-bit cache refuses on the host, beside tests/test_cache8_host.py: no kernel runs here."""
from unittest.mock import patch

import pytest
import torch

from test_cache8_host import OnCuda, batch, make, rows  # noqa: F401 (make is a fixture)


class View(OnCuda):
    """A CPU tensor that reports a CUDA device, and whose views do."""

    def view(self, *shape):
        return View(self._tensor.view(*shape))

    def __getitem__(self, i):
        return View(self._tensor[i])

    def permute(self, *dims):
        return View(self._tensor.permute(*dims))


def codes(blocks=5, heads=4, dtype=torch.float8_e4m3fn):
    return View(torch.zeros((2, blocks, 16, heads, 64), dtype=dtype))


def scale(blocks=5, heads=4, dtype=torch.float32):
    return View(torch.zeros((blocks, 2, heads), dtype=dtype))


def plane(caches, scales):
    from kvsnap_b200.dataplane import TorchBlockDataPlane
    with patch("kvsnap_b200.dataplane.CudaPool"):
        return TorchBlockDataPlane(caches, 16, 1 << 20, scales=scales)


@pytest.mark.parametrize("caches,scales,match", [
    ({"a": codes(), "b": codes()}, {"a": scale()}, "scales of b are missing"),
    ({"a": codes()}, {}, "scales of a are missing"),
    ({"a": codes()}, {"a": scale(), "c": scale()}, "scales of c, which is no registered layer"),
    ({"a": codes(), "b": codes(dtype=torch.bfloat16)}, {"a": scale(), "b": scale()}, "scales of b, which is no 8-bit"),
    ({"a": View(torch.zeros((5, 4, 16, 64), dtype=torch.uint8))}, {"a": scale()}, "no 8-bit"),
    ({"a": codes()}, {"a": scale(blocks=4)}, "as its codes are"),
    ({"a": codes()}, {"a": scale(blocks=6)}, "as its codes are"),
    ({"a": codes()}, {"a": scale(heads=2)}, "as its codes are"),
    ({"a": codes()}, {"a": scale(dtype=torch.float64)}, "as its codes are"),
    ({"a": codes()}, {"a": scale(dtype=torch.float16)}, "as its codes are"),
])
def test_scales_that_are_not_the_codes_own(caches, scales, match):
    """A block saved without its scales would be restored beside whatever its new place holds."""
    with pytest.raises(ValueError, match=match):
        plane(caches, scales)


def test_scales_beside_layers_of_16_bits_and_8_bits_without_scales():
    mixed = plane({"a": codes(), "b": codes(dtype=torch.bfloat16)}, {"a": scale()})
    assert [layer["name"] for layer in mixed.layers] == ["a.k", "a.scale", "a.v", "b.k", "b.v"]
    assert [layer["name"] for layer in plane({"a": codes()}, None).layers] == ["a.k", "a.v"]
    assert [layer["name"] for layer in plane({"a": codes(dtype=torch.uint8)}, {"a": scale()}).layers] == ["a.k", "a.scale", "a.v"]
    assert [layer["name"] for layer in plane({"a": codes(dtype=torch.bfloat16)}, {}).layers] == ["a.k", "a.v"]


@pytest.mark.parametrize("which", ["key", "value", "query"])
def test_rows_that_require_a_gradient_are_refused(make, which):    # noqa: F811
    """They would be detached without a word."""
    given = {"key": rows(), "value": rows(), "query": rows(heads=4)}
    given[which]._tensor.requires_grad_()
    rotary = OnCuda(torch.zeros((9, 32, 2)))
    cache = make()
    with pytest.raises(ValueError, match=f"{which} requires a gradient"):
        cache.append("l", given["key"], given["value"], batch(), query=given["query"], rotary=rotary)
    if which == "query":
        with pytest.raises(ValueError, match="query requires a gradient"):
            cache.attend("l", given["query"], batch())
    else:
        cache._rows(which, given["query"])
    with torch.no_grad():                                  # as a model that serves calls it
        assert cache._rows(which, given[which])


def test_check_clears_what_it_found_before_it_returns(make):    # noqa: F811
    """A call on another stream after it must not have its record cleared."""
    cache, order = make(), []

    class Word:
        def item(self):
            order.append("read")
            return 32

        def zero_(self):
            order.append("clear")

    cache.status = Word()
    with patch.object(torch.cuda, "synchronize", lambda device: order.append("wait")):
        with pytest.raises(ValueError, match="rotary"):
            cache.check()
    assert order == ["wait", "read", "clear", "wait"]
