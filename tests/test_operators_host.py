"""CPU: what the operators with gradients (imp_release_amd.ops, include/imp_hip.h) refuse before anything reaches a GPU, and their scratch sizes."""
import ctypes as C

import pytest
import torch

from imp_release_amd import _lib, ops

BAD, NOMEM = -1, -4


def desc(**over):
    d = _lib.ImpAttnDesc()
    v = dict(dtype=0, batch=2, nq=5, nk=7, heads=4, kv_heads=2, head_dim=16, scale=0.25)
    v.update({k: x for k, x in over.items() if k in v})
    for k, x in v.items():
        setattr(d, k, x)
    dh, h, kv = v['head_dim'], v['heads'], v['kv_heads']
    d.q_stride = (C.c_int64 * 3)(*over.get('q_stride', (v['nq'] * h * dh, h * dh, dh)))
    d.k_stride = d.v_stride = (C.c_int64 * 3)(v['nk'] * kv * dh, kv * dh, dh)
    return d


def message():
    return _lib.lib().imp_last_error().decode()


@pytest.mark.parametrize('over', [dict(dtype=3), dict(dtype=-1), dict(batch=0), dict(nq=0), dict(nk=0), dict(nk=-3), dict(heads=3), dict(kv_heads=0), dict(head_dim=12),
                                  dict(head_dim=136), dict(head_dim=0), dict(q_stride=(80, 18, 16)), dict(q_stride=(-320, 64, 16)), dict(batch=40000)])
def test_attention_description_refused(over):
    n = C.c_uint64()
    assert _lib.lib().imp_attn_workspace(C.byref(desc(**over)), 0, C.byref(n)) == BAD
    assert message()


def test_attention_calls_refused():
    L, d, buf = _lib.lib(), desc(), C.create_string_buffer(4096)
    at = (C.addressof(buf) + 15) // 16 * 16
    p, odd = C.c_void_p(at), C.c_void_p(at + 4)
    assert L.imp_attn_forward(C.byref(d), None, p, p, p, None, None, None, 0, 0, None) == BAD
    assert L.imp_attn_forward(C.byref(d), p, p, p, None, None, None, None, 0, 0, None) == BAD
    assert L.imp_attn_forward(C.byref(d), p, odd, p, p, None, None, None, 0, 0, None) == BAD
    assert L.imp_attn_backward(C.byref(d), p, p, p, p, None, None, p, p, p, p, p, 1 << 40, 0, None) == BAD          # no lse
    assert L.imp_attn_backward(C.byref(d), p, p, p, p, None, p, p, None, None, None, p, 1 << 40, 0, None) == BAD    # no gradient wanted
    assert L.imp_attn_backward(C.byref(d), p, p, p, p, None, p, p, p, p, None, p, 1 << 40, 0, None) == BAD          # dk without dv
    assert L.imp_attn_backward(C.byref(d), p, p, p, p, None, p, p, p, p, p, p, 8, 0, None) == NOMEM
    assert L.imp_attn_backward(C.byref(d), p, p, p, p, None, p, p, p, p, p, None, 1 << 40, 0, None) == NOMEM
    long = desc(nq=1, nk=4096)
    assert L.imp_attn_forward(C.byref(long), p, p, p, p, None, None, None, 0, 0, None) == NOMEM


def test_attention_scratch_grows_with_the_problem():
    L, n = _lib.lib(), C.c_uint64()
    sizes = []
    for nk in (64, 4096, 65536):
        assert L.imp_attn_workspace(C.byref(desc(nq=1, nk=nk)), 0, C.byref(n)) == 0
        sizes.append(n.value)
    assert sizes[0] == 0 and 0 < sizes[1] <= sizes[2]
    assert L.imp_attn_workspace(C.byref(desc(nq=100000, nk=100000, batch=16)), 1, C.byref(n)) == 0
    assert n.value >= 16 * 4 * 100000 * 4          # one float per query row


@pytest.mark.parametrize('over', [dict(dtype=7), dict(batch=0), dict(n=0), dict(channels=0), dict(groups=3), dict(groups=0), dict(batch=70000)])
def test_group_norm_sizes_refused(over):
    v = {**dict(dtype=0, batch=2, n=8, channels=32, groups=4), **over}
    n = C.c_uint64()
    assert _lib.lib().imp_group_norm_act_workspace(v['dtype'], v['batch'], v['n'], v['channels'], v['groups'], 0, C.byref(n)) == BAD and message()


def test_group_norm_calls_refused():
    L, buf = _lib.lib(), C.create_string_buffer(4096)
    at = (C.addressof(buf) + 15) // 16 * 16
    p, odd = C.c_void_p(at), C.c_void_p(at + 4)
    fwd = lambda x=p, eps=1e-3, act=0, y=p, ws=p, n=1 << 40: L.imp_group_norm_act_forward(0, 1, 4, 8, 2, x, None, None, None, eps, act, y, p, ws, n, 0, None)  # noqa: E731
    assert fwd(x=None) == BAD and fwd(y=None) == BAD and fwd(x=odd) == BAD and fwd(eps=0.0) == BAD and fwd(act=5) == BAD and fwd(act=-1) == BAD
    assert fwd(ws=None) == NOMEM and fwd(n=8) == NOMEM
    assert L.imp_group_norm_act_backward(0, 1, 4, 8, 2, p, None, None, None, 0, p, None, p, None, None, p, 1 << 40, 0, None) == BAD
    assert L.imp_group_norm_act_backward(0, 1, 4, 8, 2, p, None, None, None, 0, p, p, p, None, None, p, 8, 0, None) == NOMEM


def test_log_probs_calls_refused():
    L, buf = _lib.lib(), C.create_string_buffer(4096)
    p = C.c_void_p((C.addressof(buf) + 15) // 16 * 16)

    def fwd(dtype=0, rows=2, cols=3, ld=3, x=p, bin_=None, t=p, top=0, tv=None):
        return L.imp_log_probs_forward(dtype, rows, cols, ld, x, bin_, t, top, p, p, p, tv, tv, None, 0, 0, None)
    assert fwd(dtype=5) == BAD and fwd(rows=0) == BAD and fwd(cols=0, ld=0) == BAD and fwd(ld=2) == BAD and fwd(x=None) == BAD and fwd(t=None) == BAD
    assert fwd(top=17, tv=p) == BAD and fwd(top=-1) == BAD and fwd(top=2) == BAD and fwd(rows=1 << 31) == BAD
    assert fwd(rows=1, cols=1 << 20, ld=1 << 20) == NOMEM
    back = lambda dx=p, db=None, bin_=None, ws=None, n=0: L.imp_log_probs_backward(0, 2, 3, 3, p, bin_, p, p, p, p, p, dx, db, ws, n, 0, None)  # noqa: E731
    assert back(dx=None) == BAD and back(db=p) == BAD and back(db=p, bin_=p) == NOMEM and back(db=p, bin_=p, ws=p, n=8) == NOMEM


def test_no_cpu_path():
    x = torch.zeros(1, 2, 4, 16)
    with pytest.raises(ValueError, match='GPU'):
        ops.attention(x, x, x)
    with pytest.raises(ValueError, match='GPU'):
        ops.group_norm_act(torch.zeros(1, 4, 8), 2)
    with pytest.raises(ValueError, match='GPU'):
        ops.match_log_probs(torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError):
        ops.attention(x.double(), x, x)
    with pytest.raises(TypeError):
        ops.group_norm_act([1.0], 1)
