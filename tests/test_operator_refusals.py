"""What the operators refuse before anything reaches a GPU: wrong arguments at the C entries and tensors on the host."""
import ctypes as C

import pytest
import torch

from probtalk_amd import _lib
from probtalk_amd import train_ops as T


def refused(rc, word):
    assert rc != 0 and word in _lib.lib().pt_last_error().decode()


def test_adamw_list_refuses_host_tensors():
    t = [torch.zeros(4)]
    with pytest.raises(RuntimeError, match="GPU"):
        T.AdamWList(t, t, t)
    with pytest.raises(RuntimeError, match="GPU"):
        T.grad_norm(t, 1.0)


def test_c_entries_of_the_lists():
    L = _lib.lib()
    n, null, p = (C.c_int64 * 2)(10, 0), (C.c_void_p * 2)(None, None), (C.c_void_p * 2)(256, None)
    out = C.c_void_p(256)
    refused(L.pt_train_grad_norm(null, n, None, 2, 1.0, out, out, out, 64, None), "null tensor 0")
    refused(L.pt_train_grad_norm(p, n, None, 2, 1.0, out, out, None, 64, None), "bad argument")
    refused(L.pt_train_grad_norm(p, n, None, 2, 1.0, out, out, out, 4, None), "workspace")
    refused(L.pt_train_grad_norm(p, n, None, 2, 1.0, out, out, C.c_void_p(260), 64, None), "workspace")
    assert L.pt_train_grad_norm_workspace_bytes((C.c_int64 * 3)(1, 16384, 16385), 3) == 8 * 4
    h = (None, 1e-3, 0.9, 0.99, 1e-8, 0.0)
    refused(L.pt_train_adamw_multi(p, p, p, null, None, n, 2, 0, *h, 1, None, None, 0, None), "null tensor 0")
    refused(L.pt_train_adamw_multi(p, p, p, p, null, n, 2, 0, *h, 1, None, None, 0, None), "null tensor 0")
    refused(L.pt_train_adamw_multi(p, p, p, p, None, n, 2, 2, *h, 1, None, None, 0, None), "bad argument")
    refused(L.pt_train_adamw_multi(p, p, p, p, None, n, 2, 0, *h, 0, None, None, 0, None), "step")
    refused(L.pt_train_adamw_multi(p, p, p, p, None, n, 2, 0, *h, 0, out, None, 0, None), "scratch")
    refused(L.pt_train_moment_values(None, out, out, 4, out, out, None), "bad argument")


def test_gated_norm_refuses():
    with pytest.raises(RuntimeError, match="on the GPU"):
        T.gated_norm(torch.zeros(2, 4), pre_weight=torch.ones(4))
    L, p, odd, n = _lib.lib(), C.c_void_p(256), C.c_void_p(264), None
    fwd = lambda *a: L.pt_train_gated_norm_fwd(*a, None)  # noqa: E731
    refused(fwd(n, 4, p, 4, n, n, n, n, p, n, p, p, n, 2, 4, 2, 0, 1e-5, 0), "rows")
    refused(fwd(p, 4, p, 4, n, n, n, n, p, n, p, p, n, 0, 4, 2, 0, 1e-5, 0), "rows")
    refused(fwd(p, 9000, p, 9000, n, n, n, n, p, n, p, p, n, 2, 9000, 2, 0, 1e-5, 0), "columns")
    refused(fwd(p, 3, p, 4, n, n, n, n, p, n, p, p, n, 2, 4, 2, 0, 1e-5, 0), "stride")
    refused(fwd(p, 4, p, 4, p, n, n, n, p, n, p, p, n, 3, 4, 2, 0, 1e-5, 0), "clips")
    refused(fwd(p, 4, p, 4, n, n, n, n, p, n, p, p, n, 2, 4, 2, 2, 1e-5, 0), "kind")
    refused(fwd(p, 4, n, 0, n, n, n, n, n, n, n, n, n, 2, 4, 2, 0, 1e-5, 0), "null")
    refused(fwd(p, 4, p, 4, n, n, n, n, p, n, n, p, n, 2, 4, 2, 0, 1e-5, 0), "null")
    refused(fwd(p, 4, p, 4, n, n, n, n, p, n, p, p, odd, 2, 4, 2, 0, 1e-5, 0), "misaligned")
    bwd = lambda st, dy, dh, dx, dgate, ws, size: L.pt_train_gated_norm_bwd(p, 4, p, 4, n, n, n, n, p, st, dy, dh, dx, p, dgate, n, n, n, n, n, ws, size, 2, 4, 2, 0, 0, None)  # noqa: E731
    refused(bwd(n, p, p, p, n, p, 1 << 20), "null")
    refused(bwd(p, n, n, p, n, p, 1 << 20), "null")
    refused(bwd(p, p, p, n, n, p, 1 << 20), "null")
    refused(bwd(p, p, p, p, p, p, 1 << 20), "null")           # a gate's gradient without a gate
    refused(bwd(p, p, p, p, n, p, 0), "workspace")
    refused(bwd(p, p, p, p, n, odd, 1 << 20), "workspace")


def test_host_arrays_live_as_long_as_their_addresses():
    """Strides and pointer lists go to the C entries as addresses of arrays that nothing else refers to."""
    t = torch.zeros(5, 6, 7, 8)
    held = [T._address(T._strides(t, t[:, :1], t[:1])) for _ in range(50)]
    junk = [T._strides(t[:, ::2], t, t) for _ in range(200)]
    for a in held:
        assert list((C.c_int64 * 9).from_address(C.addressof(a))) == [336, 56, 8, 336, 0, 8, 0, 56, 8]
    assert len(junk) == 200 and T._address(None) is None


def test_window_attention_refuses():
    t = torch.zeros(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="on one GPU"):
        T.window_attention(t, t, t)
    with pytest.raises(RuntimeError, match="on one GPU"):
        T.window_attention_step(t[:, 0], t, t, torch.ones(1, dtype=torch.int32))
    L, p, odd, n = _lib.lib(), C.c_void_p(256), C.c_void_p(264), None
    st = (C.c_int64 * 9)(*([64] * 9))
    one = dict(B=1, Nq=4, Nk=4, H=2, Hk=1, D=16, left=1, right=0, sinks=0, scale=0.5, dtype=1)
    def fwd(word, q=p, lse=p, o=p, strides=st, **kw):
        refused(L.pt_attention_window_fwd(q, p, p, o, lse, strides, n, *(one | kw).values(), None), word)
    fwd("null", q=n)
    fwd("null", o=n)
    fwd("multiples", q=odd)
    fwd("multiples", strides=(C.c_int64 * 9)(*([64] * 8 + [60])))
    for kw, word in ((dict(B=0), "rows"), (dict(Nq=0), "rows"), (dict(Nq=5), "rows"), (dict(Nk=1 << 29), "rows"), (dict(B=70000), "rows"), (dict(H=3, Hk=2), "heads"),
                     (dict(Hk=0), "heads"), (dict(D=12), "dimension"), (dict(D=136), "dimension"), (dict(left=-2), "window"), (dict(sinks=129), "window"),
                     (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(dtype=2), "dtype")):
        fwd(word, **kw)
    ws = L.pt_attention_window_bwd_workspace_bytes(1, 700, 700, 2, 1, 64, 50, 0, 5)
    assert ws > 2 * 700 * 4 and L.pt_attention_window_bwd_workspace_bytes(1, 700, 700, 2, 1, 64, 50, 0, 0) == 5632
    big = (one | dict(Nq=700, Nk=700, D=64, left=50, sinks=5)).values()
    refused(L.pt_attention_window_bwd(p, p, p, p, p, p, p, p, p, st, n, *big, p, ws - 1, None), "workspace")
    refused(L.pt_attention_window_bwd(p, p, p, p, p, n, p, p, p, st, n, *big, p, ws, None), "null")
    refused(L.pt_attention_window_bwd(p, p, p, p, odd, p, p, p, p, st, n, *big, p, ws, None), "multiples")
    step = dict(B=1, N=4, H=2, Hk=1, D=16, left=1, sinks=0, scale=0.5, dtype=1)
    refused(L.pt_attention_window_step(p, p, p, p, st, n, *step.values(), p, 1 << 20, None), "null")
    refused(L.pt_attention_window_step(p, p, p, p, st, p, *(step | dict(N=0)).values(), p, 1 << 20, None), "keys")
    refused(L.pt_attention_window_step(p, p, p, p, st, p, *step.values(), p, 0, None), "workspace")
    refused(L.pt_attention_window_step(p, odd, p, p, st, p, *step.values(), p, 1 << 20, None), "multiples")


def test_gated_norm_refuses_a_bias_without_its_weight():
    """Forward would leave the bias of u out and backward count it in."""
    L, p, n = _lib.lib(), C.c_void_p(256), None
    fwd = lambda post_w, post_b, pre_w, pre_b: L.pt_train_gated_norm_fwd(p, 4, p, 4, n, n, post_w, post_b, pre_w, pre_b, p, p, n, 2, 4, 2, 0, 1e-5, 0, None)  # noqa: E731
    refused(fwd(n, p, p, p), "bias")
    refused(fwd(p, p, n, p), "bias")
    refused(L.pt_train_gated_norm_bwd(p, 4, p, 4, n, n, n, p, p, p, p, p, p, p, n, n, n, n, n, n, p, 1 << 20, 2, 4, 2, 0, 0, None), "bias")


def test_launches_of_more_threads_than_32_bits_count():
    """The largest sizes are refused before anything is launched (a grid holds less than 2^32 threads)."""
    L, p, n = _lib.lib(), C.c_void_p(256), None
    st = (C.c_int64 * 9)(*([64] * 9))
    for dtype in (0, 1):
        big = (65535, 1, 1, 512, 1, 8, 0, 0, 0, 1.0, dtype)
        refused(L.pt_attention_window_fwd(p, p, p, p, n, st, n, *big, None), "too many rows and heads")
        refused(L.pt_attention_window_bwd(p, p, p, p, p, p, p, p, p, st, n, *big, p, 1 << 40, None), "too many rows and heads")
        # the far rows of the first keys: four blocks of 32 keys for every head
        far = (65535, 129, 129, 96, 96, 8, 0, 0, 128, 1.0, dtype)
        refused(L.pt_attention_window_bwd(p, p, p, p, p, p, p, p, p, st, n, *far, p, 1 << 60, None), "too many rows and heads")
    one = (C.c_void_p * 1)(256)
    h = (None, 1e-3, 0.9, 0.99, 1e-8, 0.0)
    refused(L.pt_train_adamw_multi(one, one, one, one, one, (C.c_int64 * 1)(1 << 35), 1, 1, *h, 1, None, None, 0, None), "too many values")
    refused(L.pt_train_moment_values(p, p, p, 1 << 34, p, p, None), "bad argument")


def test_gated_norm_counts_rows_beyond_2_to_the_30():
    """A clip of rows that 32 bits hold, but not twice: 512 blocks of 32 workers, five sums of 8 columns each (256 CUs)."""
    f = _lib.lib().pt_train_gated_norm_workspace_bytes
    assert [f(n, 8, n) for n in (1 << 30, (1 << 30) + 64, (1 << 31) - 1)] == [512 * 5 * 8 * 4] * 3
    assert f(1 << 31, 8, 0) == 0
