"""What the C entry points of the attention, the gated projection and AdamW refuse before they touch a GPU."""
import ctypes as C

import pytest

from v1_glif_model_amd import _lib


def refused(rc, word=""):
    assert rc in (_lib.GLIF_EINVAL, _lib.GLIF_ENOMEM), rc
    assert word in _lib.lib().glif_last_error().decode()


def adamw(n=1, var=1 << 20, grad=1 << 21, var_dt=0, grad_dt=0, size=10, bits=32, first=1 << 22, second=1 << 23, scales=1 << 24,
          count=1 << 25, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, decay=0.0):
    k = max(n, 1)
    return _lib.lib().glif_adamw(n, (C.c_void_p * k)(*[var] * k), (C.c_int32 * k)(*[var_dt] * k), (C.c_void_p * k)(*[grad] * k),
                                 (C.c_int32 * k)(*[grad_dt] * k), (C.c_int64 * k)(*[size] * k), bits, first, second, scales, scales,
                                 count, lr, b1, b2, eps, decay, 0, None)


@pytest.mark.parametrize("kw", [dict(n=-1), dict(bits=16), dict(b1=1.0), dict(b2=-0.5), dict(b1=float("nan")), dict(eps=-1e-9),
                                dict(decay=float("nan")), dict(size=-1), dict(size=2 ** 36 + 1), dict(var_dt=3), dict(grad_dt=1),
                                dict(var_dt=1, grad_dt=2), dict(var=None), dict(first=None), dict(count=None),
                                dict(bits=8, scales=None), dict(first=(1 << 22) + 4)])
def test_adamw_refuses(kw):
    refused(adamw(**kw), "NULL" if None in kw.values() else "adamw")


@pytest.mark.parametrize("eps", [0.0, 1e-30, 9e-13, float("inf"), float("nan")])
def test_adamw_refuses_an_epsilon_that_the_squares_of_float32_do_not_reach(eps):
    """A gradient of 1e-20 has a square of 0 there: without the epsilon its step would be one of 1e-20 / 0."""
    refused(adamw(eps=eps), "epsilon")
    assert adamw(eps=1e-12, grad=None) == 0


def test_adamw_without_work():
    """No variables, no gradient, no elements: nothing to do, and no GPU needed."""
    assert adamw(n=0) == 0 and adamw(grad=None) == 0 and adamw(size=0) == 0
    refused(_lib.lib().glif_adamw_values(None, None, None, None, 255, None, None, None), "256")
    refused(_lib.lib().glif_adamw_values(None, None, None, None, 256, None, None, None), "NULL")


def attention(**kw):
    s = _lib.Attention()
    for n in ("q", "k", "v", "log_decay"):
        setattr(s, n, 1 << 20)
    s.n_ticks, s.n_batch, s.n_heads, s.n_groups, s.d_key, s.d_value = 4, 2, 4, 2, 8, 8
    for n, x in kw.items():
        setattr(s, n, x)
    return C.byref(s)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(n_ticks=-1), dict(n_ticks=2 ** 20 + 1), dict(n_batch=65536), dict(n_heads=4097),
                                dict(n_groups=3), dict(n_groups=0), dict(d_key=0), dict(d_key=129), dict(d_value=129), dict(q=None),
                                dict(log_decay=None), dict(n_batch=65535, n_heads=4096, n_groups=1)])
def test_attention_refuses(kw):
    L, g = _lib.lib(), _lib.AttentionGrad(dy=1 << 21)
    refused(L.glif_attention_fwd(attention(**kw), 1 << 22, None, None, 0, None))
    refused(L.glif_attention_bwd(attention(**kw), C.byref(g), None, 0, None))
    refused(L.glif_attention_step(attention(**kw), 1 << 22, 1 << 23, None))


def test_attention_refuses_results_whose_gradient_it_would_refuse():
    """Narrow queries and shared values, wide results: 2^24 elements from tick to tick in y, fewer in q, k and v."""
    L, wide = _lib.lib(), dict(n_batch=2 ** 13, n_heads=16, n_groups=1, d_key=8, d_value=128, q_st=2 ** 20, k_st=2 ** 16, v_st=2 ** 20)
    refused(L.glif_attention_fwd(attention(**wide), 1 << 22, None, None, 0, None), "2^24")
    assert L.glif_attention_fwd_workspace(attention(**wide)) == 0
    refused(L.glif_attention_bwd(attention(**wide), C.byref(_lib.AttentionGrad(dy=1 << 21)), None, 0, None), "2^24")
    for fits in (dict(wide, n_ticks=1), dict(wide, n_batch=2 ** 13 - 1)):   # without an output's address they get as far as that
        refused(L.glif_attention_fwd(attention(**fits), None, None, None, 0, None), "NULL")


def test_attention_refuses_missing_outputs_and_workspaces():
    L, g = _lib.lib(), _lib.AttentionGrad(dq=1 << 21)
    refused(L.glif_attention_fwd(attention(), None, None, None, 0, None), "NULL")
    refused(L.glif_attention_bwd(attention(), C.byref(g), None, 0, None), "NULL")
    refused(L.glif_attention_bwd(attention(), None, None, 0, None), "NULL")
    refused(L.glif_attention_step(attention(), 1 << 22, None, None), "NULL")
    long = attention(n_ticks=4096)
    assert L.glif_attention_fwd_workspace(long) > 0
    refused(L.glif_attention_fwd(long, 1 << 22, None, None, 0, None), "workspace")
    assert L.glif_attention_fwd(attention(n_batch=0), None, None, None, 0, None) == 0


def gated(dtype=0, bias_dtype=0, M=4, N=8, K=16, act=3, ldx=16, ldw=16, x=1 << 20, w=1 << 21, y=1 << 22):
    return _lib.lib().glif_gated_linear_fwd(x, ldx, w, ldw, None, dtype, bias_dtype, M, N, K, act, y, None, None, 0, None)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(bias_dtype=1), dict(M=-1), dict(N=2 ** 20 + 1), dict(N=-1), dict(K=2 ** 24), dict(act=4),
                                dict(ldx=2 ** 24), dict(ldw=2 ** 24), dict(x=None), dict(w=None), dict(y=None),
                                dict(N=2 ** 20, K=1024, ldw=1024)])
def test_gated_linear_refuses(kw):
    refused(gated(**kw))


def test_gated_linear_refuses_missing_workspaces_and_arguments():
    L = _lib.lib()
    assert gated(M=0) == 0 and gated(N=0) == 0
    assert L.glif_gated_linear_fwd_workspace(0, 4, 8, 2 ** 20) > 0
    refused(gated(K=2 ** 20, ldx=2 ** 20, ldw=2 ** 20), "workspace")
    a = (1 << 20, 16, 0, 0, 4, 8, 16, 3, 1 << 21, None, None, None, 0, None)
    refused(L.glif_gated_linear_bwd(1 << 22, 8, None, 1 << 23, 16, *a), "NULL")
    refused(L.glif_gated_linear_bwd(1 << 22, 8, 1 << 24, 1 << 23, 16, *a), "workspace")
    refused(L.glif_gated_linear_bwd(None, 8, 1 << 24, 1 << 23, 16, *a), "NULL")
