"""Arguments that the operators between a layer's projections refuse, before anything touches a device."""
import math

import numpy as np
import pytest

import sptmm_amd as sp


def attention_args(**changes):
    a = dict(q=4096, k=8192, v=12288, out=16384, q_stride=256, k_stride=128, v_stride=128, out_stride=256, kv_rows=64, q_start=64, kv_start=64, kv_len=64, batch=2, total_q=10,
             max_q=5, max_kv=32, q_heads=4, kv_heads=2, head_dim=64, type=sp.X_F16, scale=0.125)
    a.update(changes)
    return sp.AttentionArgs(**a)


@pytest.mark.parametrize("changes", [
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q_start=None), dict(kv_start=None), dict(kv_len=None), dict(type=0), dict(type=sp.X_F32), dict(batch=-1), dict(total_q=-1),
    dict(max_q=-1), dict(max_kv=-1), dict(kv_rows=-1), dict(kv_rows=(1 << 30) + 1), dict(q_heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(q_heads=65536, kv_heads=1), dict(head_dim=0),
    dict(head_dim=4), dict(head_dim=60), dict(head_dim=264), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(scale=1e30), dict(q_stride=255), dict(q_stride=248),
    dict(k_stride=120), dict(v_stride=132), dict(out_stride=252), dict(out_stride=258), dict(k_stride=(1 << 22) + 8), dict(q=4098), dict(k=8200), dict(v=12290), dict(out=16388),
    dict(q_start=66), dict(kv_start=65), dict(kv_len=67), dict(total_q=1 << 29, q_heads=4), dict(total_q=(1 << 27) + 1, q_heads=4), dict(batch=1 << 25)])
def test_attention_refuses(changes):
    with pytest.raises(sp.SptmmError) as e:
        sp.attention(attention_args(**changes), 4096, 1 << 40)
    assert e.value.code == -1 and str(e.value)


def test_attention_wants_its_workspace():
    a = attention_args(batch=1, total_q=1, max_q=1, max_kv=10000, kv_rows=10000)
    n = sp.attention_workspace_bytes(a)
    assert n > 0
    for ws, size in ((None, n), (4096, n - 1), (4096, 0), (4100, n)):
        with pytest.raises(sp.SptmmError):
            sp.attention(a, ws, size)
    assert sp.attention_workspace_bytes(attention_args(head_dim=60)) == 0
    # few sequences in very many rows: not split, as one launch of the join holds less than 2^24 rows
    assert sp.attention_workspace_bytes(attention_args(batch=1, total_q=1 << 22, max_q=1, max_kv=10000, kv_rows=10000)) == 0


def test_attention_of_nothing_is_a_call_without_work():
    sp.attention(attention_args(batch=0), None, 0)
    sp.attention(attention_args(total_q=0, q=None, out=None), None, 0)
    with pytest.raises(AttributeError):
        sp.AttentionArgs(head_size=64)
    with pytest.raises(TypeError):
        sp.attention(heads_args(), None, 0)
    with pytest.raises(TypeError):
        sp.heads_norm_rotate(attention_args())


def heads_args(**changes):
    a = dict(q=4096, k=8192, v=12288, q_stride=256, k_stride=128, v_stride=128, in_type=sp.X_F32, out_type=sp.X_F16, q_out=4096, k_out=4096, v_out=4096, q_out_stride=256,
             k_out_stride=128, v_out_stride=128, tokens=3, q_heads=4, kv_heads=2, head_dim=64, kv_capacity=3, q_gain=4096, k_gain=4096, eps=1e-5)
    a.update(changes)
    return sp.HeadsArgs(**a)


@pytest.mark.parametrize("changes", [
    dict(q=None), dict(k=None), dict(q_out=None), dict(k_out=None), dict(v_out=None), dict(in_type=0), dict(in_type=4), dict(out_type=sp.X_F32), dict(tokens=-1), dict(q_heads=-1),
    dict(q_heads=0, kv_heads=0), dict(q_heads=70000, q_stride=1 << 30, q_out_stride=1 << 30), dict(head_dim=0), dict(head_dim=63), dict(head_dim=258), dict(q_stride=255), dict(k_stride=127),
    dict(v_stride=1), dict(q_out_stride=255), dict(k_out_stride=127), dict(v_out_stride=127), dict(kv_capacity=-1), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf), dict(q=4098),
    dict(q_out=4097), dict(positions=4098), dict(kv_rows=4097), dict(q_gain=4098)])
def test_heads_refuses(changes):
    with pytest.raises(sp.SptmmError) as e:
        sp.heads_norm_rotate(heads_args(**changes))
    assert e.value.code == -1 and str(e.value)


def test_heads_refuses_a_rotation_wider_than_the_head():
    with pytest.raises(sp.SptmmError):
        sp.heads_norm_rotate(heads_args(rotation=sp.Rotation(np.ones(33))))
    sp.heads_norm_rotate(heads_args(tokens=0, rotation=sp.Rotation(np.ones(32))))  # no tokens: nothing to do


def test_rotations():
    r = sp.Rotation([2 * math.pi / 4, -2 * math.pi / 4, 2 * math.pi * 7.5, 0.0], interleaved=True)
    assert r.pairs == 4 and r.interleaved == 1
    turns = [r.turns[j] / 2.0 ** 64 for j in range(4)]
    assert np.allclose(turns, [0.25, 0.75, 0.5, 0.0], atol=1e-14)
    for bad in (np.ones(129), [math.nan], [math.inf]):
        with pytest.raises(sp.SptmmError):
            sp.Rotation(bad)
    assert sp.Rotation().pairs == 0


@pytest.mark.parametrize("a", [(0, 16, 1, 1, 1), (16, 0, 1, 1, 1), (24, 16, 1, 1, 1), (16, 24, 1, 1, 1), (1 << 21, 16, 1, 1, 1), (16, 16, 0, 1, 1), (16, 16, 3, 1, 1), (16, 16, 1, 0, 1), (16, 16, 1, 65537, 1),
                               (16, 16, 1, 1, 0), (16, 16, 1, 1, 257), (-16, 16, 1, 1, 1)])
def test_adapters_create_refuses(a):
    with pytest.raises(sp.SptmmError) as e:
        sp.Adapters(*a)
    assert e.value.code == -1


def test_argument_blocks_keep_what_they_point_at():
    """A block is kept from call to call: a buffer made for one of its fields must not be freed under it."""
    import ctypes as C
    import gc
    import weakref

    def buffer():
        b = object.__new__(sp.DeviceBuffer)  # (no device needed: nothing allocated, nothing to free)
        b.ptr, b.nbytes = C.c_void_p(), 0
        return b, weakref.ref(b)

    for args, field, other in ((heads_args(), "q_gain", "positions"), (attention_args(), "kv_len", "kv_start")):
        b, seen = buffer()
        setattr(args, field, b)
        setattr(args, other, b)
        del b
        gc.collect()
        assert seen() is not None
        setattr(args, other, None)
        gc.collect()
        assert seen() is not None and getattr(args, other) is None
        second, later = buffer()
        setattr(args, field, second)
        del second
        gc.collect()
        assert seen() is None and later() is not None  # replaced: the first is let go
        setattr(args, field, 64)
        gc.collect()
        assert later() is None and getattr(args, field) == 64
    a = heads_args(rotation=sp.Rotation([0.5, 0.25]))
    a.tokens = 5
    gc.collect()
    assert a.rotation.contents.pairs == 2
    a.rotation = None
    assert not a.rotation


@pytest.mark.parametrize("sizes", [dict(batch=1, total_q=1, max_q=1), dict(batch=7, total_q=7, max_q=1), dict(batch=3, total_q=20, max_q=8), dict(batch=2, total_q=150, max_q=100),
                                   dict(batch=1, total_q=60, max_q=60, q_heads=40, kv_heads=8, q_stride=2560, out_stride=2560, k_stride=512, v_stride=512)])
def test_a_workspace_for_the_longest_cache_serves_the_shorter_ones(sizes):
    """max_kv grows from call to call while a cache fills: what the largest asks for is enough all the way."""
    needs = [sp.attention_workspace_bytes(attention_args(max_kv=n, kv_rows=70000, **sizes)) for n in [*range(1, 3000, 7), *range(3000, 70000, 997)]]
    assert needs[-1] > 0 and needs == sorted(needs)


def test_copies_of_argument_blocks_can_be_changed():
    a = attention_args()
    for b in (sp.AttentionArgs.from_buffer_copy(a), sp.AttentionArgs()):
        b.batch, b.q = 7, 8192
        assert (b.batch, b.q) == (7, 8192)
    assert a.batch == 2 and a.q == 4096
