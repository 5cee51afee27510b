"""What the operators of mi355x-attention.h refuse, on a host-only context:
arguments are checked before the device is reached, and a call that passes the
checks fails at the gate."""
import ctypes

import pytest

import mi355x
from mi355x import BF16, EHIP, EINVAL, EUNSUPPORTED, F16, F32, OK


@pytest.fixture(scope="module")
def host():
    with mi355x.Context(mi355x.DEVICE_HOST_ONLY) as c:
        yield c


A = 1 << 20  # an aligned address that no check may touch


def pool(**over):
    f = dict(type=F16, n_kv_heads=2, head_dim=64, page_tokens=16, n_pages=8, k=A, v=A, page_stride=2048,
             token_stride=128, head_stride=64)
    f.update(over)
    return mi355x.KvPool(**f)


def plan(**over):
    f = dict(n_seqs=2, page_tokens=16, table_cols=4, n_free=8, table_stride=4, n_rows=6, cached=A, added=A,
             block_table=A, free_pages=A, free_head=A, free_head_out=A, row_offsets=A, kv_lens=A, positions=A,
             slots=A, status=None)
    f.update(over)
    return mi355x.KvPlanArgs(**f)


def rope(p=None, **over):
    p = pool() if p is None else p
    f = dict(n_rows=3, n_heads=4, n_kv_heads=2, head_dim=64, rot_dim=64, rope_mode=0, in_type=F32, out_type=F16,
             eps=1e-6, q=A, k=A, v=A, q_stride=256, k_stride=128, v_stride=128, positions=A, inv_freq=A, q_out=A + 64,
             q_out_stride=256, pool=mi355x.pointer(p) if p else None, slots=A)
    f.update(over)
    return mi355x.QkNormRopeArgs(**f)


def attn(p=None, **over):
    f = dict(n_rows=3, n_seqs=2, n_heads=4, max_added=2, q=A, q_stride=256, pool=mi355x.pointer(p or pool()),
             row_offsets=A, kv_lens=A, block_table=A, table_cols=4, table_stride=4, scale=0.125, causal=1, out=A,
             out_type=F16, out_stride=256, workspace=A, workspace_bytes=1 << 40)
    f.update(over)
    return mi355x.PagedAttentionArgs(**f)


def rc(host, fn, args):
    return getattr(host.lib, fn)(host.h, ctypes.byref(args))


@pytest.mark.parametrize("fn,make", [("mi355x_kv_plan", plan), ("mi355x_qk_norm_rope", rope),
                                     ("mi355x_paged_attention", attn)])
def test_good_arguments_reach_the_gate(host, fn, make):
    assert rc(host, fn, make()) == EHIP
    assert mi355x.last_error().startswith(fn + ": hipErrorNoDevice")
    assert getattr(host.lib, fn)(host.h, None) == EINVAL and "null" in mi355x.last_error()
    assert getattr(host.lib, fn)(None, ctypes.byref(make())) == EINVAL


@pytest.mark.parametrize("over", [
    dict(n_seqs=-1), dict(n_seqs=65537), dict(page_tokens=0), dict(page_tokens=24), dict(page_tokens=1 << 17),
    dict(n_rows=-1), dict(n_rows=2 ** 31), dict(table_cols=-1), dict(n_free=-1), dict(table_stride=3),
    dict(table_stride=-1), dict(table_stride=2 ** 31), dict(cached=None), dict(added=None), dict(block_table=None),
    dict(free_pages=None), dict(free_head=None), dict(free_head_out=None), dict(row_offsets=None),
    dict(kv_lens=None), dict(positions=None), dict(slots=None), dict(cached=A + 2), dict(slots=A + 4),
    dict(status=A + 1)])
def test_plan_refuses(host, over):
    assert rc(host, "mi355x_kv_plan", plan(**over)) == EINVAL
    assert mi355x.last_error().startswith("mi355x_kv_plan: ")


def test_plan_allows(host):
    for over in (dict(n_seqs=0, cached=None, added=None, kv_lens=None, block_table=None),
                 dict(n_rows=0, positions=None, slots=None), dict(n_free=0, free_pages=None),
                 dict(table_cols=0, block_table=None), dict(status=A)):
        assert rc(host, "mi355x_kv_plan", plan(**over)) == EHIP, over


POOLS = [dict(type=F32), dict(type=7), dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=60), dict(page_tokens=0),
         dict(page_tokens=12), dict(n_pages=-1), dict(n_pages=2 ** 31), dict(k=None), dict(v=None), dict(k=A + 8),
         dict(page_stride=-8), dict(token_stride=4), dict(head_stride=2 ** 31 + 8)]


@pytest.mark.parametrize("over", POOLS)
def test_pools_refused(host, over):
    assert rc(host, "mi355x_qk_norm_rope", rope(pool(**over))) == EINVAL
    assert rc(host, "mi355x_paged_attention", attn(pool(**over))) == EINVAL


@pytest.mark.parametrize("over", [
    dict(n_rows=-1), dict(n_rows=2 ** 31), dict(n_heads=-1), dict(n_heads=65537), dict(head_dim=63), dict(head_dim=0),
    dict(head_dim=1026), dict(head_dim=32), dict(n_kv_heads=1), dict(rot_dim=66), dict(rot_dim=3), dict(rot_dim=-2),
    dict(rope_mode=2), dict(in_type=2), dict(out_type=F32), dict(out_type=BF16), dict(out_type=5),
    dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(q=None), dict(q_out=None), dict(k=None),
    dict(v=None), dict(slots=None), dict(positions=None), dict(inv_freq=None), dict(q_stride=255), dict(k_stride=127),
    dict(v_stride=1), dict(q_out_stride=8), dict(q_stride=2 ** 41), dict(q=A + 2), dict(q_out=A + 1),
    dict(q_bias=A + 2), dict(k_norm=A + 1), dict(slots=A + 4), dict(q_out=A)])
def test_rope_refuses(host, over):
    assert rc(host, "mi355x_qk_norm_rope", rope(**over)) == EINVAL
    assert mi355x.last_error().startswith("mi355x_qk_norm_rope: ")


def test_rope_without_a_pool(host):
    ok = dict(pool=None, slots=None, v=None, k_out=A + 64, k_out_stride=128)
    assert rc(host, "mi355x_qk_norm_rope", rope(**ok)) == EHIP
    for over in (dict(k_out=None), dict(k_out_stride=64), dict(k_out=A), dict(k_out=A + 1)):
        assert rc(host, "mi355x_qk_norm_rope", rope(**{**ok, **over})) == EINVAL, over
    assert rc(host, "mi355x_qk_norm_rope", rope(**{**ok, "out_type": F32, "q_out": A, "k_out": A})) == EHIP


def test_rope_of_no_rows_is_done(host):
    assert rc(host, "mi355x_qk_norm_rope", rope(n_rows=0, q=None, k=None, v=None)) == OK
    assert rc(host, "mi355x_qk_norm_rope", rope(rot_dim=0, positions=None, inv_freq=None)) == EHIP


@pytest.mark.parametrize("over", [
    dict(n_rows=-1), dict(n_rows=2 ** 31), dict(n_seqs=-1), dict(n_seqs=65537), dict(n_heads=0), dict(n_heads=3),
    dict(max_added=-1), dict(q=None), dict(out=None), dict(row_offsets=None), dict(kv_lens=None),
    dict(block_table=None), dict(table_cols=-1), dict(table_stride=3), dict(table_stride=2 ** 31),
    dict(table_cols=2 ** 27, table_stride=2 ** 27), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(softcap=-1.0), dict(softcap=float("inf")), dict(window=-1), dict(out_type=BF16), dict(out_type=3),
    dict(q_stride=255), dict(q_stride=260), dict(out_stride=128), dict(out_stride=260), dict(q=A + 8),
    dict(out=A + 2), dict(kv_lens=A + 2)])
def test_attention_refuses(host, over):
    assert rc(host, "mi355x_paged_attention", attn(**over)) == EINVAL
    assert mi355x.last_error().startswith("mi355x_paged_attention: ")


@pytest.mark.parametrize("hd", [8, 32, 72, 120, 192, 512])
def test_head_sizes_that_are_not_computed(host, hd):
    p = pool(head_dim=hd, token_stride=2 * hd, head_stride=hd, page_stride=32 * hd)
    assert rc(host, "mi355x_paged_attention", attn(p, q_stride=4 * hd, out_stride=4 * hd)) == EUNSUPPORTED
    n = ctypes.c_size_t()
    assert host.lib.mi355x_paged_attention_workspace(host.h, 4, 2, hd, ctypes.byref(n)) == EUNSUPPORTED
    assert host.lib.mi355x_paged_attention_workspace(host.h, 4, 3, 64, ctypes.byref(n)) == EINVAL
    assert host.lib.mi355x_paged_attention_workspace(host.h, 4, 2, 64, None) == EINVAL
    assert host.lib.mi355x_paged_attention_workspace(host.h, 4, 2, 64, ctypes.byref(n)) == EHIP


@pytest.mark.parametrize("rows,seqs,heads,kv,code", [
    (65536, 65536, 128, 128, EUNSUPPORTED), (65536, 65536, 127, 127, EHIP), (2 ** 30 - 128, 1, 2, 1, EUNSUPPORTED),
    (2 ** 30 - 256, 1, 1, 1, EHIP), (2 ** 26, 1, 16, 16, EUNSUPPORTED)])
def test_as_many_blocks_as_a_launch_takes(host, rows, seqs, heads, kv, code):
    p = pool(n_kv_heads=kv, token_stride=64 * kv, page_stride=1024 * kv)
    a = attn(p, n_rows=rows, n_seqs=seqs, n_heads=heads, q_stride=64 * heads, out_stride=64 * heads)
    assert rc(host, "mi355x_paged_attention", a) == code


def test_attention_of_no_rows_is_done(host):
    assert rc(host, "mi355x_paged_attention", attn(n_rows=0, q=None, out=None)) == OK
    assert rc(host, "mi355x_paged_attention", attn(n_seqs=0, row_offsets=None)) == OK


@pytest.mark.parametrize("fn,make", [("mi355x_kv_plan", plan), ("mi355x_qk_norm_rope", rope),
                                     ("mi355x_paged_attention", attn)])
def test_injected_faults(host, fn, make):
    mi355x.inject_fault(fn, mi355x.HIP_ERROR_LAUNCH_FAILURE)
    try:
        assert rc(host, fn, make()) == EHIP
        assert "[injected]" in mi355x.last_error()
    finally:
        mi355x.inject_fault(None)
