"""Calls of the penalties that their C entry has to refuse before it launches anything."""

from __future__ import annotations

import ctypes as C

import pytest

from insitu_b200 import _lib


def refused(rows=1, vocab=5, dtype=0, logits=0, out=0, **fields):
    """ins_penalize's status over host memory, none of which a refused call reads; logits and out are `logits`
    and `out` bytes from an aligned address."""
    memory = C.create_string_buffer(512)
    base = (C.addressof(memory) + 15) // 16 * 16
    args = _lib.PenaltiesArgs(**{k: base + v if k not in SIZES else v for k, v in fields.items()})
    return _lib.lib().ins_penalize(rows, vocab, base + logits, dtype, vocab, base + out, vocab, C.byref(args), None)


SIZES = ("history", "histories", "n_drafted")
OF_4 = ("lengths", "prompts", "of", "repetition", "presence", "frequency", "bias", "mask")


@pytest.mark.parametrize("name", OF_4 + ("tokens", "drafted"))
def test_buffers_that_are_not_aligned_to_their_elements_are_refused(name):
    """The kernel loads whole elements; an address between two would be a fault on the device."""
    for off in (1, 2, 3) if name in OF_4 else (1, 4, 7):
        assert refused(history=1, histories=1, n_drafted=1, **{name: off}) == _lib.INS_EINVAL, off
    assert b"aligned" in _lib.lib().ins_last_error()


def test_logits_and_results_that_are_not_aligned_are_refused():
    for dtype, offs in ((0, (1, 2, 3)), (1, (1, 3)), (2, (1, 3))):
        for off in offs:
            assert refused(dtype=dtype, logits=off) == _lib.INS_EINVAL
            assert refused(dtype=dtype, out=off) == _lib.INS_EINVAL


def test_tokens_that_together_would_reach_the_bit_beside_a_count_are_refused():
    """A token said 2^31 times would read as one of the prompt, never said."""
    assert refused(histories=1, tokens=0, drafted=0, history=1 << 30, n_drafted=1 << 30) == _lib.INS_EBADLEN


@pytest.mark.gpu
def test_a_result_over_another_argument_is_refused():
    """A row of the result that is another row's bias, or all rows', would be written while it is read."""
    torch = pytest.importorskip("torch")
    from insitu_b200 import Penalties
    x, wide = torch.randn((4, 3001), device="cuda"), torch.randn((9, 3001), device="cuda")
    tokens = torch.randint(0, 3001, (4, 20), device="cuda")
    p = Penalties(repetition=[1.0, 1.5, 1.1, 1.2])
    want = p(x, tokens, bias=wide[0])
    for kw in (dict(bias=wide[0], out=wide[:4]), dict(bias=wide[3], out=wide[:4]), dict(bias=wide[1:5], out=wide[:4]),
               dict(bias=wide[:4], out=wide[1:5]), dict(mask=wide.view(torch.int32)[2, :94], out=wide[:4])):
        with pytest.raises(ValueError):
            p(x, tokens, **kw)
    long = torch.zeros((4, 6002), dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        p(x, long[:, :7], out=long.view(torch.float32)[:, :3001])
    assert torch.equal(p(x, tokens, bias=wide[0], out=wide[1:5]), want)
    assert Penalties()(x[:0], bias=wide[0], out=wide[:0]).shape == (0, 3001)


@pytest.mark.gpu
def test_arguments_beside_the_result_in_wider_rows_are_not_over_it():
    """Columns [0, 3001) of a buffer's rows hold the result, others a bias of each row or of all."""
    torch = pytest.importorskip("torch")
    from insitu_b200 import Penalties
    x = torch.randn((4, 3001), device="cuda")
    tokens = torch.randint(0, 3001, (4, 20), device="cuda")
    p = Penalties(repetition=[1.0, 1.5, 1.1, 1.2])
    buffer = torch.randn((4, 6010), device="cuda")
    for bias in (buffer[:, 3001:6002], buffer[:, 3009:], buffer[2, 3005:6006]):
        want = p(x, tokens, bias=bias.clone())
        assert torch.equal(p(x, tokens, bias=bias, out=buffer[:, :3001]), want)
    for bias in (buffer[:, 3000:6001], buffer[1, 3000:6001], buffer.flatten()[3010:6011]):
        with pytest.raises(ValueError):
            p(x, tokens, bias=bias, out=buffer[:, :3001])
