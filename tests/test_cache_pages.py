"""Pages of the 4-bit latent cache: refusals and bookkeeping that need no GPU."""
import ctypes

import pytest
import torch

from palu_amd import _lib
from palu_amd.kernel import paged


def _host_pool(N=4, G=2, P=16, Rk=32, Rv=64, **change):
    t = dict(k_codes=torch.zeros(N, G, P, Rk // 2, dtype=torch.uint8), k_meta=torch.zeros(N, G, P, 2, dtype=torch.float16),
             v_codes=torch.zeros(N, G, P, Rv // 2, dtype=torch.uint8), v_meta=torch.zeros(N, G, P, 2, dtype=torch.float16))
    t.update(change)
    return paged.PagePool(**t)


def test_there_is_no_cpu_path():
    pool = _host_pool()
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(TypeError, match="no CPU fallback"):
        paged.paged_append(pool, torch.zeros(1, 2, 32).half(), torch.zeros(1, 2, 64).half(), i.view(1, 1), i, i)
    with pytest.raises(TypeError, match="no CPU fallback"):
        paged.paged_copy(pool, [0], [1])
    with pytest.raises(TypeError, match="no CPU fallback"):
        paged.paged_attn(torch.zeros(1, 8, 128).half(), i, pool, i.view(1, 1), i)
    with pytest.raises(TypeError, match="no CPU fallback"):
        paged.prepare_paged_b(torch.zeros(8, 32, 128).half(), 2)


@pytest.mark.parametrize("change,err", [
    (dict(k_meta=torch.zeros(4, 2, 16, 3, dtype=torch.float16)), ValueError),
    (dict(v_codes=torch.zeros(4, 2, 32, 32, dtype=torch.uint8)), ValueError),
    (dict(k_codes=torch.zeros(4, 2, 16, 16)), TypeError),
    (dict(k_codes=torch.zeros(2, 16, 16, dtype=torch.uint8)), ValueError)])
def test_pools_that_do_not_fit_are_refused(change, err):
    with pytest.raises(err):
        paged.paged_copy(_host_pool(**change), [0], [1])


def _args(**over):
    """Arguments of palu_paged_attn_q4 with pointers that are never followed (every call here is refused before the launch)."""
    a = dict(q=16, sq_b=256, sq_h=128, bfrag=16, kc=16, km=16, vc=16, vm=16, table=16, st_b=4, max_pages=4, lens=16, qpos=0, inv=16,
             ctx=16, ws=16, B=1, H=2, G=1, D=128, P=64, n_pages=4, Rk=64, Rv=64, scale=0.1, stream=0)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(D=64), -2), (dict(P=24), -2), (dict(P=8), -2), (dict(Rk=36), -2), (dict(Rk=264), -2), (dict(Rv=520), -2), (dict(Rv=0), -2),
    (dict(H=3, G=2), -1), (dict(n_pages=0), -1), (dict(max_pages=1 << 25, P=64), -1), (dict(q=0), -1), (dict(ws=0), -1),
    (dict(lens=0), -1), (dict(B=-1), -1), (dict(B=1 << 20), -1)])
def test_attention_entry_refuses(over, code):
    assert _lib.lib.palu_paged_attn_q4(*_args(**over)) == code
    assert b"paged_attn" in _lib.lib.palu_last_error()


def test_empty_calls_are_no_calls():
    """nothing to do: no pointer is looked at and nothing is launched"""
    assert _lib.lib.palu_paged_attn_q4(*_args(B=0, q=0, kc=0, lens=0)) == 0
    assert _lib.lib.palu_paged_copy(0, 0, 0, 0, 0, 0, 0, 1, 4, 1, 16, 32, 32, 0) == 0
    assert _lib.lib.palu_paged_append_q4(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 1, 1, 0, 0, 0, 1, 16, 4, 32, 32, 0) == 0


@pytest.mark.parametrize("over,code", [(dict(P=17), -2), (dict(P=8), -2), (dict(Rk=12), -2), (dict(n=-1), -1), (dict(layers=0), -1),
                                       (dict(kc=8), -1), (dict(src=0), -1)])
def test_copy_entry_refuses(over, code):
    a = dict(kc=16, km=16, vc=16, vm=16, src=16, dst=16, n=1, layers=1, n_pages=4, G=1, P=16, Rk=32, Rv=32, stream=0)
    a.update(over)
    assert _lib.lib.palu_paged_copy(*a.values()) == code and b"paged_copy" in _lib.lib.palu_last_error()


@pytest.mark.parametrize("over,code", [(dict(P=48), -2), (dict(Rk=12), -2), (dict(Rv=520), -2), (dict(k=8), -1), (dict(sk_t=4), -1),
                                       (dict(seq=0), -1), (dict(n_pages=0), -1), (dict(T=-1), -1)])
def test_append_entry_refuses(over, code):
    a = dict(k=16, sk_t=32, sk_g=32, v=16, sv_t=32, sv_g=32, kc=16, km=16, vc=16, vm=16, table=16, st_b=1, B=1, max_pages=1, seq=16,
             pos=16, T=1, G=1, P=16, n_pages=4, Rk=32, Rv=32, stream=0)
    a.update(over)
    assert _lib.lib.palu_paged_append_q4(*a.values()) == code and b"paged_append" in _lib.lib.palu_last_error()


def test_layout_of_b_has_a_size_only_where_the_kernel_takes_it():
    size = _lib.lib.palu_paged_b_bytes
    assert size(32, 8, 128) >= 32 * 128 * 128 * 2 and size(10, 5, 40) >= 10 * 40 * 128 * 2 and size(8, 1, 256) > 0
    assert size(32, 5, 128) == 0 and size(32, 8, 264) == 0 and size(32, 8, 36) == 0 and size(0, 1, 64) == 0
    assert ctypes.sizeof(ctypes.c_size_t) == 8
