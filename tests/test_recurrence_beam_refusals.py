"""What the recurrence and the beam search refuse, on the host and before any launch."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def fr():
    from fast_rnnt_b200 import build
    build.build()
    import fast_rnnt_b200
    return fast_rnnt_b200


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_recurrence_arguments(fr):
    for args in [(z(2, 3), z(2, 3)),                                      # no time axis
                 (z(2, 3, 4), z(2, 3, 5)), (z(2, 3, 4), z(2, 3, 4, dtype=torch.float16)),
                 (z(2, 3, 4), z(2, 3, 4))]:                               # CPU tensors
        with pytest.raises(AssertionError):
            fr.gated_recurrence(*args)
    with pytest.raises(TypeError):
        fr.gated_recurrence(z(2, 3, 4, dtype=torch.int32), z(2, 3, 4, dtype=torch.int32))


def test_step_arguments(fr):
    x, p = z(2, 3, 4), z(2, 3, dtype=torch.int64)
    for args in [(x, z(2, 3, 5), x), (x, x, z(2, 3, 4, dtype=torch.float64)), (x, x, z(2, 2, 4)),
                 (x, x, z(3, 5, 4), p), (x, x, z(2, 5, 4), z(2, 2, dtype=torch.int64)),
                 (x, x, z(2, 5, 4), z(2, 3)), (x, x, x)]:
        with pytest.raises(AssertionError):
            fr.gated_recurrence_step(*args)


def test_beam_arguments(fr):
    logits, scores = z(2, 3, 9), z(2, 3)
    for args in [(z(2, 9), scores, 3), (logits, z(2, 4), 3), (logits, z(2, 3, dtype=torch.float64), 3),
                 (z(2, 0, 9), z(2, 0), 3), (logits, scores, 3)]:
        with pytest.raises(AssertionError):
            fr.beam_select(*args)
    with pytest.raises(TypeError):
        fr.beam_select(logits.double(), scores, 3)
    for states, parents in [([z(2, 3, 4)], z(2, 3)), ([z(2, 3, 4)], z(2, 3, dtype=torch.int64))]:
        with pytest.raises(AssertionError):
            fr.beam_reorder(states, parents)


def test_c_abi_checks(fr):
    from fast_rnnt_b200 import _lib
    lib, n = _lib.lib(), ctypes.c_longlong
    one = ctypes.c_void_p(16)

    def refused(name, *args, code=-1, text=b""):
        assert getattr(lib, name)(*args) == code, name
        assert text in lib.frnnt_last_error(), lib.frnnt_last_error()

    seq = lambda dtype, B, T, D, x=one: ("frnnt_recurrence_forward", dtype, x, n(0), n(0), one, n(0), n(0), None,  # noqa: E731
                                         None, one, one, None, B, T, D, None)
    refused(*seq(9, 1, 1, 1), text=b"dtype")
    refused(*seq(0, 1, -1, 1), text=b"sizes")
    refused(*seq(0, 1, 1, 1, None), text=b"NULL")
    assert lib.frnnt_recurrence_forward(*seq(0, 0, 5, 5)[1:]) == 0
    back = lambda dtype, saved: ("frnnt_recurrence_backward", dtype, one, n(0), n(0), one, n(0), n(0), None, saved,  # noqa: E731
                                 None, n(0), n(0), None, one, one, None, 1, 400, 4, None)
    refused(*back(-1, one), text=b"dtype")
    refused(*back(0, None), text=b"NULL")
    refused("frnnt_recurrence_step", 0, one, n(4), one, n(4), one, None, None, one, n(2), 1, 1, 4, None,
            text=b"overwrite")
    assert lib.frnnt_recurrence_saved_bytes(7, 1, 1, 1) == 0
    select = lambda dtype, B, K, V, beam, done=None, blank=0: (  # noqa: E731
        "frnnt_beam_select", dtype, one, n(V), n(V), one, done, blank, one, one, one, one, B, K, V, beam, None)
    refused(*select(1, 1, 2, 5, 2), text=b"dtype")
    refused(*select(0, 1, 0, 5, 2), text=b"sizes")
    refused(*select(0, 1, 2, 5, 0), code=-2, text=b"beam")
    refused(*select(0, 1, 2, 5, 33), code=-2, text=b"beam")
    refused(*select(0, 1, 1025, 5, 2), code=-2, text=b"beams")
    refused(*select(0, 1, 1000, 1 << 22, 2), code=-2, text=b"2^31")
    refused(*select(0, 1, 2, 5, 2, one, 5), text=b"termination")
    refused("frnnt_beam_reorder", -1, None, one, 1, 1, 1, None, text=b"sizes")
    refused("frnnt_beam_reorder", 1, None, one, 1, 1, 1, None, text=b"NULL")
    for to, text in ((16, b"in place"), (0, b"NULL")):
        refused("frnnt_beam_reorder", 1, (n * 5)(16, to, 16, 16, 16), one, 1, 1, 1, None, text=text)
