"""Adam's scalars are used in f32: what f32 does not hold is refused, on the
host and before any launch."""
import ctypes

import pytest

import bindcraft2_amd as b

P = 4096  # an address that no refused call reads
MAX = 3.4028234663852886e38  # f32's largest


@pytest.fixture(params=[64, 100000], ids=["one workgroup", "several"])
def adam(request):
    one = lambda t, v: (t * 1)(v)  # noqa: E731
    at = [one(ctypes.c_void_p, k * 1000 * P) for k in range(1, 5)]
    p, g, m, v = at
    t = one(ctypes.c_int, 0)
    h = b.lib().bc2n_adam_list(1, one(ctypes.c_int64, request.param), p, t, g, t, m, v, p, m, v)
    assert h
    yield lambda lr=0.1, b1=0.9, eps=1e-8, wd=0.0, t=1, mx=0.0, scalars=None: (
        b.lib().bc2n_adam_step(None, h, lr, b1, 0.99, eps, wd, t, mx, scalars, None, P))
    b.lib().bc2n_list_free(h)


@pytest.mark.parametrize("scalars,text", [
    ({"eps": 1e-46}, b"eps"),  # rounds to 0: 0 / 0 where a gradient has always been zero
    ({"eps": 2.0 ** -150}, b"eps"),  # half of f32's smallest step: to even, 0
    ({"eps": 1e39}, b"eps"),
    ({"eps": float("inf")}, b"eps"),
    ({"eps": float("nan")}, b"eps"),
    ({"eps": 1e-46, "scalars": P}, b"eps"),
    ({"wd": float("inf")}, b"weight_decay"),
    ({"wd": float("inf"), "lr": 0.0}, b"weight_decay"),
    ({"wd": float("inf"), "scalars": P}, b"weight_decay"),
    ({"wd": float("nan")}, b"weight_decay"),
    ({"lr": 1e39}, b"learning rate"),
    ({"lr": -1e39}, b"learning rate"),
    ({"lr": MAX}, b"learning rate"),  # over 1 - 0.9 it is past f32
    ({"lr": 1e30, "wd": 1e10}, b"learning rate"),
], ids=str)
def test_scalars_past_f32(adam, scalars, text):
    assert adam(**scalars) != 0
    assert text in b.lib().bc2n_last_error(), b.lib().bc2n_last_error()
