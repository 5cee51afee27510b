"""What the operators of mi355x-layer.h refuse, on a host-only context:
arguments are checked before the device is reached, and a call that passes the
checks fails at the gate."""
import ctypes

import numpy as np
import pytest

import layer_ref
import mi355x
from mi355x import BF16, EHIP, EINVAL, F16, F32, OK


@pytest.fixture(scope="module")
def host():
    with mi355x.Context(mi355x.DEVICE_HOST_ONLY) as c:
        yield c


A = 1 << 20  # an aligned address that no check may touch


def make(cls, f, over):
    return cls(**{**f, **over})


def norm(**over):
    return make(mi355x.NormQ8Args, dict(n_rows=3, n=100, type=F16, x=A, x_stride=100, residual_type=F32, eps=1e-6,
                                        residual=2 * A, residual_stride=104, residual_out=3 * A,
                                        residual_out_stride=100, norm=4 * A, q=5 * A, q_stride=100, scales=6 * A), over)


def swiglu(**over):
    return make(mi355x.SwigluQ8Args, dict(n_rows=3, n=100, type=F32, gate=A, gate_stride=200, up=A + 400,
                                          up_stride=200, q=5 * A, q_stride=100, scales=6 * A), over)


def matmul(**over):
    return make(mi355x.MatmulQ8Args, dict(n_rows=3, n_out=70, k=96, x=A, x_stride=96, x_scales=2 * A, w=3 * A,
                                          w_stride=112, w_scales=4 * A, bias=5 * A, out=6 * A, out_type=BF16,
                                          out_stride=70, workspace=7 * A, workspace_bytes=1 << 40), over)


def logprobs(**over):
    return make(mi355x.LogprobsArgs, dict(n_rows=3, n_vocab=1000, type=BF16, logits=A, stride=1001, scale=1.0,
                                          n_tokens=2, tokens=2 * A, token_logprobs=3 * A, entropy=4 * A, n_top=5,
                                          top_tokens=5 * A, top_logprobs=6 * A, workspace=7 * A,
                                          workspace_bytes=1 << 40), over)


CALLS = {"mi355x_norm_q8": norm, "mi355x_swiglu_q8": swiglu, "mi355x_matmul_q8": matmul,
         "mi355x_logprobs": logprobs}


def rc(host, fn, args):
    return getattr(host.lib, fn)(host.h, ctypes.byref(args))


@pytest.mark.parametrize("fn", CALLS)
def test_good_arguments_reach_the_gate(host, fn):
    assert rc(host, fn, CALLS[fn]()) == EHIP
    assert mi355x.last_error().startswith(fn + ": hipErrorNoDevice")
    assert getattr(host.lib, fn)(host.h, None) == EINVAL and "null" in mi355x.last_error()
    assert getattr(host.lib, fn)(None, ctypes.byref(CALLS[fn]())) == EINVAL


@pytest.mark.parametrize("fn", CALLS)
def test_no_rows_are_no_work(host, fn):
    gone = {f: None for f, t in CALLS[fn]()._fields_ if t is ctypes.c_void_p}
    assert rc(host, fn, CALLS[fn](n_rows=0, **gone)) == OK


@pytest.mark.parametrize("fn", ["mi355x_matmul_q8_workspace", "mi355x_logprobs_workspace"])
def test_workspace_sizes_need_a_device(host, fn):
    n = ctypes.c_size_t()
    assert getattr(host.lib, fn)(host.h, ctypes.byref(n)) == EHIP
    assert getattr(host.lib, fn)(host.h, None) == EINVAL and getattr(host.lib, fn)(None, ctypes.byref(n)) == EINVAL


REFUSED = [
    ("mi355x_norm_q8", [
        dict(n_rows=-1), dict(n_rows=2 ** 31), dict(n=0), dict(n=65537), dict(type=2), dict(residual_type=2),
        dict(eps=-1.0), dict(eps=float("inf")), dict(eps=float("nan")), dict(x=None), dict(x=A + 1), dict(x_stride=99),
        dict(x_stride=-1), dict(x_stride=2 ** 41), dict(residual=None), dict(residual=A + 2), dict(residual_stride=99),
        dict(residual_out=A + 2), dict(residual_out_stride=99), dict(residual_out=2 * A),
        dict(residual_out=A, residual_out_stride=100), dict(residual_out=A, residual_out_stride=104, residual_type=F16),
        dict(norm=A + 2), dict(q=None), dict(q_stride=99), dict(scales=None), dict(scales=A + 1)]),
    ("mi355x_swiglu_q8", [
        dict(n_rows=-1), dict(n=0), dict(n=65537), dict(type=3), dict(gate=None), dict(up=None), dict(gate=A + 2),
        dict(up=A + 1), dict(gate_stride=99), dict(up_stride=99), dict(q=None), dict(q_stride=50), dict(scales=None),
        dict(scales=A + 3)]),
    ("mi355x_matmul_q8", [
        dict(n_rows=-1), dict(n_rows=2 ** 24 + 1), dict(n_out=-1), dict(n_out=2 ** 24 + 1), dict(k=0), dict(k=8),
        dict(k=100), dict(k=131072), dict(out_type=2), dict(x=None), dict(w=None), dict(x=A + 8), dict(w=A + 4),
        dict(x_stride=80), dict(w_stride=80), dict(x_stride=104), dict(w_stride=104), dict(x_scales=None),
        dict(w_scales=None), dict(x_scales=A + 2), dict(w_scales=A + 1), dict(bias=A + 2), dict(out=None),
        dict(out=A + 1), dict(out_stride=69)]),
    ("mi355x_logprobs", [
        dict(n_rows=-1), dict(n_vocab=0), dict(n_vocab=2 ** 30 + 1), dict(type=2), dict(scale=0.0), dict(scale=-1.0),
        dict(scale=float("inf")), dict(scale=float("nan")), dict(n_tokens=-1), dict(n_tokens=65537), dict(n_top=-1),
        dict(n_top=65), dict(logits=None), dict(logits=A + 1), dict(stride=999), dict(tokens=None),
        dict(tokens=A + 2), dict(token_logprobs=None), dict(token_logprobs=A + 1), dict(entropy=A + 2),
        dict(top_tokens=None), dict(top_logprobs=None), dict(top_tokens=A + 1), dict(top_logprobs=A + 2)]),
]


@pytest.mark.parametrize("fn,over", [(fn, o) for fn, all_ in REFUSED for o in all_])
def test_refuses(host, fn, over):
    assert rc(host, fn, CALLS[fn](**over)) == EINVAL
    assert mi355x.last_error().startswith(fn + ": ")


@pytest.mark.parametrize("fn,over", [
    ("mi355x_norm_q8", dict(residual=None, residual_out=None, residual_type=99)),
    ("mi355x_norm_q8", dict(residual_out=None)), ("mi355x_norm_q8", dict(norm=None)),
    ("mi355x_norm_q8", dict(residual_out=2 * A, residual_out_stride=104)),
    ("mi355x_norm_q8", dict(residual_out=A, residual_out_stride=100, residual_type=F16)),
    ("mi355x_norm_q8", dict(n_rows=1, x_stride=0, residual_stride=0, residual_out_stride=0, q_stride=0)),
    ("mi355x_norm_q8", dict(n=65536, x_stride=65536, residual_stride=65536, residual_out_stride=65536,
                            q_stride=65536)),
    ("mi355x_swiglu_q8", dict(q=5 * A + 1)),
    ("mi355x_matmul_q8", dict(bias=None)), ("mi355x_matmul_q8", dict(k=131056, x_stride=131056, w_stride=131056)),
    ("mi355x_matmul_q8", dict(out=A + 2)),
    ("mi355x_logprobs", dict(entropy=None)), ("mi355x_logprobs", dict(n_top=0, top_tokens=None, top_logprobs=None)),
    ("mi355x_logprobs", dict(n_tokens=0, tokens=None, token_logprobs=None)),
    ("mi355x_logprobs", dict(n_vocab=1, stride=1, n_top=64))])
def test_allows(host, fn, over):
    assert rc(host, fn, CALLS[fn](**over)) == EHIP


def test_nothing_asked_is_no_work(host):
    assert rc(host, "mi355x_logprobs", logprobs(n_tokens=0, n_top=0, entropy=None, logits=None)) == OK
    assert rc(host, "mi355x_matmul_q8", matmul(n_out=0, w=None)) == OK


def test_the_reference_rounds_ties_to_even():
    c, s, _ = layer_ref.codes_of(np.array([[381, 1.5 * 3, 2.5 * 3, -0.5 * 3, -1.5 * 3, 0.5 * 3]]))
    assert c.tolist() == [[127, 2, 2, 0, -2, 0]] and np.all(s == 3)
    c, s, _ = layer_ref.codes_of(np.array([[0.0, 0.0], [1.0, np.inf], [np.nan, 1.0]]))
    assert not c.any() and s[0] == 0 and np.isnan(s[1:]).all()


def test_scales_past_their_limits(host):
    for scale, want in [(2.0 ** 100, EHIP), (2.0 ** -100, EHIP), (2.0 ** 101, EINVAL), (2.0 ** -101, EINVAL)]:
        assert rc(host, "mi355x_logprobs", logprobs(scale=scale)) == want


def test_products_too_large(host):
    wide = dict(out_stride=2 ** 24)
    for over, want in [
            (dict(wide, n_rows=1024, n_out=2 ** 24), mi355x.EUNSUPPORTED), (dict(wide, n_rows=1023, n_out=2 ** 24), EHIP),
            (dict(n_rows=64 * 65535 + 1, x_stride=2 ** 23 + 16), mi355x.EUNSUPPORTED),
            (dict(n_rows=64 * 65535 + 1, w_stride=2 ** 23 + 16), mi355x.EUNSUPPORTED),
            (dict(n_rows=64 * 65535, x_stride=2 ** 23 + 16), EHIP),
            (dict(n_rows=64 * 65535 + 1, x_stride=2 ** 23), EHIP)]:
        assert rc(host, "mi355x_matmul_q8", matmul(**over)) == want
