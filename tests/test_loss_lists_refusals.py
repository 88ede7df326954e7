"""The refusals of the log-probability and gradient-list entry points, which
are made on the host before any GPU call."""
import ctypes

import bindcraft2_amd as b

F32, F16, BF16 = 0, 1, 2
P = 4096  # an address that no refused call reads


def refused(status, text):
    assert status != 0 and text in b.lib().bc2n_last_error(), b.lib().bc2n_last_error()


def fwd(dtype=F32, x=P, ld=64, rows=4, v=64, t=P, bits=64, top=0, logp=P, entropy=P, tl=None, ti=None,
        save=P, work=P):
    return b.lib().bc2n_logprobs_fwd(None, dtype, x, ld, rows, v, t, bits, top, logp, entropy, tl, ti,
                                     save, work)


def bwd(x=P, ld=64, rows=4, v=64, t=P, bits=32, top=0, ti=None, save=P, g=P, e=None, h=None, d=2 * P, dld=64):
    return b.lib().bc2n_logprobs_bwd(None, BF16, x, ld, rows, v, t, bits, top, ti, save, g, e, h, d, dld)


def test_logprobs_refusals():
    refused(fwd(dtype=3), b"dtype")
    refused(fwd(rows=-1), b"rows")
    refused(fwd(rows=1 << 31), b"rows")
    refused(fwd(v=0), b"classes")
    refused(fwd(v=1 << 29, ld=1 << 29), b"classes")
    refused(fwd(ld=63), b"stride")
    refused(fwd(bits=16), b"i32 or i64")
    refused(fwd(x=None), b"null")
    refused(fwd(t=None), b"targets")
    refused(fwd(top=33, tl=P, ti=P), b"top")
    refused(fwd(top=-1), b"top")
    refused(fwd(v=3, top=4, tl=P, ti=P), b"top")
    refused(fwd(top=2, tl=P), b"null")
    refused(fwd(x=P + 2), b"unaligned")
    refused(fwd(t=P + 4), b"unaligned")
    refused(fwd(save=P + 8), b"unaligned")
    refused(fwd(work=P + 8), b"unaligned")
    refused(bwd(d=P + 1), b"unaligned")
    refused(bwd(save=P + 4), b"unaligned")
    refused(bwd(d=None), b"null")
    refused(bwd(dld=63), b"stride")
    refused(bwd(d=P, ld=64, dld=65), b"in place")
    refused(bwd(d=P + 2), b"overlaps")
    refused(bwd(d=P + 2 * 64 * 3 + 2 * 63), b"overlaps")  # the last row's last class
    refused(bwd(x=P + 2 * 64, d=P), b"overlaps")
    refused(bwd(ld=200, d=P + 2 * 63, dld=200), b"overlaps")
    refused(bwd(ld=200, d=P + 2 * 150, dld=200), b"overlaps")  # into the next row
    refused(bwd(ld=200, d=P + 2 * 100, dld=201), b"overlaps")
    refused(bwd(ld=200, d=P + 2 * 64, dld=200, save=None), b"null")  # columns beside: taken
    refused(bwd(save=None), b"null")
    refused(bwd(t=None), b"targets")
    refused(bwd(h=P), b"top_index")
    refused(bwd(h=P, top=2), b"top_index")
    refused(b.lib().bc2n_logprobs_grad(None, F32, P, 64, 4, 64, None, 32, P, None, None, P, 2 * P, 64, P),
            b"targets")
    assert b.lib().bc2n_logprobs_work_bytes(7, 4, 64, 0) == 0
    assert b"dtype" in b.lib().bc2n_last_error()
    assert b.lib().bc2n_logprobs_save_bytes(10) == 160
    assert b.lib().bc2n_logprobs_work_bytes(F16, 9, 8192, 32) == 0


def ptrs(*v):
    return (ctypes.c_void_p * len(v))(*v)


def grad_list(grads, sizes, types=None, out=None):
    n = len(grads)
    return b.lib().bc2n_grad_list(n, ptrs(*grads), (ctypes.c_int64 * n)(*sizes),
                                  (ctypes.c_int * n)(*(types or [F32] * n)), ptrs(*out) if out else None)


def no_list(handle, text):
    assert handle is None and text in b.lib().bc2n_last_error(), b.lib().bc2n_last_error()


def test_list_refusals():
    """Short lists live on the host, so their checks need no GPU."""
    L = b.lib()
    no_list(grad_list([P], [-1]), b"negative")
    no_list(grad_list([None], [4]), b"null")
    no_list(grad_list([P + 2], [4]), b"unaligned")
    no_list(grad_list([P], [4], [5]), b"dtype")
    no_list(grad_list([P], [4], out=[None]), b"null")
    no_list(grad_list([P, P], [4, 4], out=[P, P]), b"shares memory")
    no_list(grad_list([P, P + 12], [4, 4], out=[P, P + 12]), b"shares memory")
    no_list(grad_list([P, 2 * P], [4, 4], out=[2 * P, 3 * P]), b"shares memory")
    no_list(grad_list([P], [8], out=[P + 4]), b"shares memory")
    no_list(L.bc2n_grad_list(-1, None, None, None, None), b"null")
    h = grad_list([P, P + 16, None], [4, 4, 0], out=[P, P + 16, None])  # neighbours
    assert h and L.bc2n_list_work_bytes(h) == 0  # a small list needs none
    L.bc2n_list_free(h)
    h = grad_list([P, P + 400000, None], [100000, 4, 0], out=[P, P + 400000, None])
    assert h and L.bc2n_list_work_bytes(h) > 0
    refused(L.bc2n_grad_clip(None, h, 0.0, P, P), b"max_norm")
    refused(L.bc2n_grad_clip(None, h, float("nan"), P, P), b"max_norm")
    refused(L.bc2n_grad_clip(None, h, 1.0, P, None), b"null")
    refused(L.bc2n_grad_norm(None, h, None, P), b"null")
    refused(L.bc2n_adam_step(None, h, 0.1, 0.9, 0.99, 1e-8, 0, 1, 0, None, None, P), b"parameters")
    assert L.bc2n_list_free(h) == 0 and L.bc2n_list_free(None) == 0
    h = grad_list([P, P], [4, 4])  # the same gradient twice, only read
    refused(L.bc2n_grad_clip(None, h, 1.0, P, P), b"no outputs")
    refused(L.bc2n_grad_norm(None, None, P, P), b"not a list")
    L.bc2n_list_free(h)


def test_adam_refusals():
    L = b.lib()
    one = lambda t, v: (t * 1)(v)  # noqa: E731

    def make(p=P, g=2 * P, m=3 * P, v=4 * P, po=P, mo=3 * P, vo=4 * P, pt=F32, gt=F32, n=64,
             far=1):
        p, g, m, v, po, mo, vo = (x and x * far for x in (p, g, m, v, po, mo, vo))
        return L.bc2n_adam_list(1, one(ctypes.c_int64, n), ptrs(p), one(ctypes.c_int, pt), ptrs(g),
                                one(ctypes.c_int, gt), ptrs(m), ptrs(v), ptrs(po), ptrs(mo), ptrs(vo))

    no_list(make(pt=3), b"dtype")
    no_list(make(m=None), b"null")
    no_list(make(vo=3 * P), b"shares memory")
    no_list(make(g=P), b"shares memory")
    no_list(make(m=3 * P + 2, mo=3 * P + 2), b"unaligned")
    h = make(pt=BF16, gt=F16, p=P + 2, po=P + 2)
    assert h and L.bc2n_list_work_bytes(h) == 0
    L.bc2n_list_free(h)
    h = make(n=100000, far=100)
    assert h

    def step(lr=0.1, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, t=1, mx=0.0, work=P):
        return L.bc2n_adam_step(None, h, lr, b1, b2, eps, wd, t, mx, None, None, work)

    refused(step(b1=1.0), b"betas")
    refused(step(b2=-0.5), b"betas")
    refused(step(eps=0.0), b"eps")
    refused(step(wd=-1.0), b"weight_decay")
    refused(step(t=0), b"step")
    refused(step(lr=float("inf")), b"step")
    refused(step(mx=float("nan")), b"max_norm")
    refused(step(work=None), b"null")
    refused(L.bc2n_grad_clip(None, h, 1.0, P, P), b"no outputs")
    L.bc2n_list_free(h)
