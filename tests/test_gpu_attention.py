"""GPU: sptmm_attention against the definition in 64 bits (tests/operators64.py holds it and the error bounds)."""
import numpy as np
import pytest

import operators64 as op
import sptmm_amd as sp

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    return sp.device_init(0)


class Call:
    """One attention call: inputs from a seed, strides and gaps as asked, buffers on the device."""

    def __init__(self, seed, nq, nk, heads, dim, t, packed=False, tail=0, gap=5, pad=0, max_q=None, max_kv=None, scale=None, edit=None, sharp=1.5):
        r = np.random.default_rng(seed)
        hq, hkv = heads
        self.t, self.dim, self.hq, self.hkv = t, dim, hq, hkv
        self.q_start = np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)
        self.kv_len = np.asarray(nk, np.int32)
        self.kv_start = self.q_start[:-1].copy() if packed else np.concatenate([[0], np.cumsum(np.asarray(nk) + gap)])[:-1].astype(np.int32)
        self.rows = max(1, int((self.kv_start + self.kv_len).max()) + (0 if packed else gap))
        self.total = int(self.q_start[-1]) + tail
        self.scale = scale or op.softmax_scale(dim)
        q, k, v = r.standard_normal((self.total, hq, dim)) * sharp, r.standard_normal((self.rows, hkv, dim)), r.standard_normal((self.rows, hkv, dim))
        if edit:
            edit(self, q, k, v)
        self.q, self.k, self.v = (op.narrow(x, t)[1] for x in (q, k, v))
        wide = [np.full((len(x), x.shape[1] * dim + pad), np.nan, np.float32) for x in (q, k, v)]  # what lies between rows is never read
        for w, x in zip(wide, (q, k, v)):
            w[:, : x.shape[1] * dim] = x.reshape(len(x), -1)
        self.bufs = [sp.DeviceBuffer.from_numpy(op.narrow(w, t)[0]) for w in wide]
        self.out_pad = pad
        self.before, _ = op.narrow(r.standard_normal((self.total, hq * dim + self.out_pad)), t)
        self.out = sp.DeviceBuffer.from_numpy(self.before)
        ints = [sp.DeviceBuffer.from_numpy(x) for x in (self.q_start, self.kv_start, self.kv_len)]
        self.bufs += ints
        self.args = sp.AttentionArgs(q=self.bufs[0], k=self.bufs[1], v=self.bufs[2], out=self.out, q_stride=hq * dim + pad, k_stride=hkv * dim + pad, v_stride=hkv * dim + pad,
                                     out_stride=hq * dim + self.out_pad, kv_rows=self.rows, q_start=ints[0], kv_start=None if packed else ints[1],
                                     kv_len=None if packed else ints[2], batch=len(nq), total_q=self.total, max_q=max(nq) if max_q is None else max_q,
                                     max_kv=max(nk) if max_kv is None else max_kv, q_heads=hq, kv_heads=hkv, head_dim=dim, type=op.CODE[t], scale=self.scale)

    def run(self, stream=None):
        n = sp.attention_workspace_bytes(self.args)
        self.ws_bytes = n
        self.ws = sp.DeviceBuffer(n + 256)
        self.ws.fill(0xFF)  # NaN everywhere: nothing may be read that was not written
        sp.attention(self.args, self.ws, n, stream)
        sp.device_sync()
        assert (self.ws.to_numpy(np.uint8, n + 256)[n:] == 0xFF).all()
        self.got = self.out.to_numpy(op.buffer_type(self.t), self.before.shape)
        return self

    def check(self):
        want = op.attention(self.q, self.k, self.v, self.q_start, self.kv_start, self.kv_len, self.scale, self.t)
        got = op.widen(self.got, self.t)
        for row in range(self.total):
            mine = got[row, : self.hq * self.dim].reshape(self.hq, self.dim)
            if row not in want:
                assert (self.got[row].view(np.uint16) == self.before[row].view(np.uint16)).all(), "row %d behind the last sequence was written" % row
                continue
            o, e = want[row]
            fine = np.isfinite(o)
            assert (np.isnan(mine) == np.isnan(o)).all(), ("NaN", row)
            assert (mine[~fine & ~np.isnan(o)] == o[~fine & ~np.isnan(o)]).all(), ("Inf", row)
            off = np.abs(mine - o)[fine]
            assert (off <= e[fine]).all(), (row, float((off / e[fine]).max()))
            if self.out_pad:
                assert (self.got[row, self.hq * self.dim:].view(np.uint16) == self.before[row, self.hq * self.dim:].view(np.uint16)).all()
        return self

    def free(self):
        for b in self.bufs + [self.out, self.ws]:
            b.free()


def one(*a, **k):
    print("attention", a, {x: y for x, y in k.items() if x != "edit"}, flush=True)
    c = Call(*a, **k).run()
    c.check().free()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [8, 64, 72, 80, 128, 136, 256])
def test_prompts_of_every_width(dim, t):
    one(1, [1, 33, 0, 130, 7], [1, 33, 0, 130, 7], (4, 2), dim, t, packed=True)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("heads", [(1, 1), (5, 5), (6, 2), (20, 5), (12, 1), (40, 1)])
def test_heads_per_group(heads, t):
    one(2, [70, 3], [70, 3], heads, 64, t, packed=True)
    one(3, [1, 1, 1], [70, 3, 129], heads, 64, t)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257])
def test_prompt_lengths(n):
    one(4, [n], [n], (2, 1), 128, "bf16", packed=True)


@pytest.mark.parametrize("m", [0, 1, 31, 32, 33, 64, 127, 128, 129, 255, 256, 257, 1000])
def test_one_token_against_a_cache(m):
    one(5, [1], [m], (20, 5), 128, "f16")
    one(6, [1, 1], [m, 3], (8, 8), 64, "bf16", tail=2)


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_ragged_decode_batch_with_empty_caches_and_a_long_one(t):
    nk = [0, 1, 2, 700, 0, 33, 5000, 128, 127]
    one(7, [1] * len(nk), nk, (20, 5), 128, t, tail=3)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_chunks_of_prompts_against_longer_and_shorter_caches(dim):
    # the second sequence's cache is shorter than its chunk (its first rows see nothing), the third's is empty
    one(8, [40, 50, 9, 1, 100], [500, 20, 0, 77, 1300], (4, 2), dim, "bf16", tail=1)
    one(9, [3, 5, 0, 2], [300, 4, 10, 2], (8, 2), dim, "f16")


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [40, 128, 256])
def test_equal_shares_of_unequal_chunks(dim, t):
    """Shares that end within a tile, shares of several short tiles, rows that see nothing of a part or nothing at all."""
    one(30, [40, 130, 0, 9, 1, 300], [3000, 20, 500, 0, 5000, 1700], (6, 2), dim, t, tail=2, pad=8)


def test_equal_shares_of_many_sequences_and_of_one_tile():
    r = np.random.default_rng(31)
    one(31, [int(x) for x in r.integers(0, 20, 150)], [int(x) for x in r.integers(0, 1500, 150)], (8, 1), 64, "bf16")
    one(32, [9], [40000], (4, 1), 64, "f16")  # 79 parts


@pytest.mark.parametrize("nq,nk,heads", [([2100, 300], [2100, 300], (2, 1)), ([900, 900], [2300, 2049], (3, 3)), ([513], [513], (4, 4))])
def test_equal_shares_of_prompts(nq, nk, heads):
    one(33, nq, nk, heads, 64, "f16", max_kv=5000)


@pytest.mark.parametrize("what", [np.inf, np.nan])
def test_what_is_not_finite_stays_with_its_rows_across_shares(what):
    def edit(c, q, k, v):
        v[c.kv_start[0] + 1990, 0, 3] = what  # seen by the last rows of the first sequence only
        k[c.kv_start[1] + 1995, 1] = what

    one(34, [60, 50], [2000, 2000], (4, 2), 64, "bf16", edit=edit)


def test_rows_strides_and_gaps():
    one(10, [5, 60], [40, 77], (4, 2), 64, "f16", pad=8, tail=4)
    one(11, [1, 1], [400, 77], (4, 2), 128, "bf16", pad=24, tail=4)


def test_many_sequences():
    r = np.random.default_rng(0)
    nk = [int(x) for x in r.integers(0, 40, 150)]
    one(12, [1] * 150, nk, (4, 4), 64, "f16")
    one(13, nk, nk, (2, 1), 64, "bf16", packed=True)


@pytest.mark.parametrize("max_q,max_kv", [(0, 0), (1, 1), (1, 100000), (100000, 1), (3, 600), (1 << 30, 1 << 30)])
def test_results_do_not_depend_on_the_hints_being_right(max_q, max_kv):
    one(14, [1, 40, 3, 129], [900, 700, 3, 129], (4, 2), 128, "bf16", max_q=max_q, max_kv=max_kv)


@pytest.mark.parametrize("scale", [1e-6, 0.01, 3.0])
@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_flat_and_sharp_scores(scale, t):
    one(15, [1, 90], [600, 90], (4, 2), 64, t, scale=scale)


def test_scores_that_climb_and_fall_along_the_keys():
    def edit(c, q, k, v):
        k[:] = k * 0.1 + np.linspace(-3, 3, len(k))[:, None, None]
        q[0::2] = np.abs(q[0::2])
        q[1::2] = -np.abs(q[1::2])
    one(16, [2, 70], [2000, 400], (4, 2), 64, "f16", edit=edit)
    one(17, [1, 1], [3000, 2000], (4, 2), 128, "bf16", edit=edit)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_what_is_not_finite_reaches_the_rows_that_see_it_only(what, t):
    # rows behind the caches and between them
    def outside(c, q, k, v):
        live = np.zeros(len(k), bool)
        for s, n in zip(c.kv_start, c.kv_len):
            live[s:s + n] = True
        k[~live], v[~live] = what, what
    one(18, [1, 40, 1], [33, 40, 300], (4, 2), 64, t, edit=outside)

    # a value in the middle of a prompt: rows before it are as if it were not there
    def inside(c, q, k, v):
        v[37, 0, 5] = what
        v[150, 1, 63] = what
    one(19, [200], [200], (4, 2), 64, t, packed=True, edit=inside)
    one(20, [150, 4], [180, 70], (4, 2), 128, t, edit=inside)
    one(21, [2, 5], [38, 152], (4, 2), 64, t, edit=inside)


def test_a_key_of_minus_infinity_scores_takes_no_weight():
    def edit(c, q, k, v):
        q[:] = np.abs(q) + 0.1
        k[10:40, 0] = -np.inf
        k[0, :] = -np.inf
    one(22, [100], [100], (2, 1), 64, "bf16", packed=True, edit=edit)
    one(23, [1], [300], (2, 1), 64, "f16", edit=edit)


def test_cache_rows_behind_four_gigabytes():
    """A cache whose last rows lie more than 2^32 bytes and 2^31 elements behind its first, read through a wide row stride."""
    dim, hkv, stride, n = 64, 1, 1 << 22, 600
    rows = n
    big = sp.DeviceBuffer(2 * stride * rows)  # 5 GB; only the rows themselves are written
    r = np.random.default_rng(3)
    k, kv64 = op.narrow(r.standard_normal((rows, hkv * dim)), "bf16")
    host = np.zeros((rows, dim), np.uint16)
    host[:] = k
    import ctypes as C
    for i in range(rows):
        rc = sp.lib().sptmm_memcpy_h2d(C.c_void_p(big.ptr.value + 2 * stride * i), host[i].ctypes.data_as(C.c_void_p), C.c_size_t(2 * dim))
        assert rc == 0
    q, q64 = op.narrow(r.standard_normal((2, 2 * dim)), "bf16")
    qb, out = sp.DeviceBuffer.from_numpy(q), sp.DeviceBuffer(2 * q.size)
    ints = [sp.DeviceBuffer.from_numpy(np.array(x, np.int32)) for x in ([0, 1, 2], [0, 530], [600, 70])]
    a = sp.AttentionArgs(q=qb, k=big, v=big, out=out, q_stride=2 * dim, k_stride=stride, v_stride=stride, out_stride=2 * dim, kv_rows=rows, q_start=ints[0], kv_start=ints[1],
                         kv_len=ints[2], batch=2, total_q=2, max_q=1, max_kv=600, q_heads=2, kv_heads=1, head_dim=dim, type=2, scale=0.125)
    for max_q in (1, 200):  # both forms
        print("long cache, max_q", max_q, flush=True)
        a.max_q = max_q
        n_ws = sp.attention_workspace_bytes(a)
        ws = sp.DeviceBuffer(n_ws + 16)
        sp.attention(a, ws, n_ws)
        sp.device_sync()
        got = op.widen(out.to_numpy(np.uint16, (2, 2, dim)), "bf16")
        want = op.attention(q64.reshape(2, 2, dim), kv64.reshape(rows, 1, dim), kv64.reshape(rows, 1, dim), [0, 1, 2], [0, 530], [600, 70], 0.125, "bf16")
        for row in (0, 1):
            assert (np.abs(got[row] - want[row][0]) <= want[row][1]).all()
        ws.free()
    for b in [big, qb, out] + ints:
        b.free()


def test_a_captured_call_follows_its_buffers():
    """Three replays with new queries, keys and lengths in the captured buffers, eager work between them."""
    st = sp.Stream()
    c = Call(30, [1, 1, 1], [900, 40, 0], (20, 5), 128, "bf16", max_kv=2000, gap=600)
    n = sp.attention_workspace_bytes(c.args)
    c.ws = sp.DeviceBuffer(n + 256)
    with sp.Graph(st) as g:
        sp.attention(c.args, c.ws, n, st)
    r = np.random.default_rng(5)
    for rep in range(3):
        print("replay", rep, flush=True)
        qb, c.q = op.narrow(r.standard_normal(c.q.shape), "bf16")
        kb, c.k = op.narrow(r.standard_normal(c.k.shape), "bf16")
        c.kv_len = np.array([1500 - 300 * rep, 41 + rep, rep], np.int32)
        c.bufs[0].upload(qb)
        c.bufs[1].upload(kb)
        c.bufs[5].upload(c.kv_len)
        g.launch(st)
        st.sync()
        first = c.out.to_numpy(np.uint16, c.before.shape)
        c.got = first
        c.check()
        c.out.upload(c.before)
        sp.attention(c.args, c.ws, n, st)  # the program's own eager work
        st.sync()
        assert (c.out.to_numpy(np.uint16, c.before.shape) == first).all()
    g.destroy()
    c.free()
    st.destroy()


def test_lengths_that_lead_out_of_the_buffers_are_cut():
    """The arrays on the device are data: whatever they hold, nothing outside the buffers is read or written (the rows' values are
    not specified then; the call returns and the device goes on working)."""
    c = Call(31, [4, 4, 4], [20, 20, 20], (4, 2), 64, "f16", tail=2)
    c.bufs[3].upload(np.array([0, 9, 3, 1 << 30], np.int32))
    c.bufs[4].upload(np.array([-5, 1 << 30, 40], np.int32))
    c.bufs[5].upload(np.array([1 << 30, 10, 1 << 30], np.int32))
    c.run()
    c.free()
    one(32, [4, 4], [20, 20], (4, 2), 64, "f16")


def test_a_captured_call_of_shares_follows_its_lengths():
    """How the work is shared out is found on the device: a replay with other lengths gives what a fresh call gives."""
    st = sp.Stream()
    c = Call(40, [60, 90, 20], [1500, 700, 40], (6, 2), 128, "bf16", max_kv=2500, gap=1200, max_q=120)
    n = sp.attention_workspace_bytes(c.args)
    assert n > 0
    c.ws = sp.DeviceBuffer(n + 256)
    with sp.Graph(st) as g:
        sp.attention(c.args, c.ws, n, st)
    for rep, (first, length) in enumerate((([0, 60, 150, 170], [2400, 700, 0]), ([0, 1, 120, 170], [3, 1900, 900]), ([0, 0, 170, 170], [0, 650, 5]))):
        print("replay", rep, flush=True)
        c.q_start, c.kv_len = np.array(first, np.int32), np.array(length, np.int32)
        c.bufs[3].upload(c.q_start)
        c.bufs[5].upload(c.kv_len)
        c.ws.fill(0xFF)
        g.launch(st)
        st.sync()
        c.got = got = c.out.to_numpy(np.uint16, c.before.shape)
        c.check()
        c.out.upload(c.before)
        sp.attention(c.args, c.ws, n, st)
        st.sync()
        assert (c.out.to_numpy(np.uint16, c.before.shape) == got).all()
    g.destroy()
    c.free()
    st.destroy()


@pytest.mark.parametrize("dim", [64, 256])
def test_shares_of_lengths_that_lead_out_of_the_buffers(dim):
    c = Call(41, [90, 60, 70], [2000, 900, 20], (6, 2), dim, "f16", tail=2)
    assert sp.attention_workspace_bytes(c.args) > 0
    c.bufs[3].upload(np.array([0, 200, 3, 1 << 30], np.int32))
    c.bufs[4].upload(np.array([-5, 1 << 30, 40], np.int32))
    c.bufs[5].upload(np.array([1 << 30, 10, 1 << 30], np.int32))
    c.run()
    c.free()
    one(42, [4, 4], [20, 20], (4, 2), 64, "f16")


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("below", [3, 12, 18, 22, 26])
@pytest.mark.parametrize("nq", [1, 40])
def test_many_small_weights_beside_a_large_one(nq, below, t):
    """One key of weight 1 and value 0, thousands of weight 2^-below and value 1: small weights count in both sums alike."""
    def edit(c, q, k, v):
        q[:], k[:], v[:] = 0.0, 0.0, 1.0
        q[:, :, 0], k[5, :, 0], v[5] = 1.0, below, 0.0

    one(43, [nq], [9000], (4, 1), 64, t, edit=edit, scale=float(np.log(2.0)))


def test_a_row_of_one_key_is_its_value():
    c = Call(44, [1, 1, 1, 70], [1, 1, 1, 70], (4, 2), 128, "bf16", packed=True).run()
    v = op.narrow(c.v, "bf16")[0].reshape(c.rows, 2, 128)
    for row in range(4):  # (the fourth is the first query of the last sequence)
        got = c.got[row].reshape(4, 128)
        assert all((got[h].view(np.uint16) == v[row, h // 2].view(np.uint16)).all() for h in range(4)), row
    c.free()


@pytest.mark.parametrize("nq", [[1, 1], [40, 3]])
def test_no_cache_at_all(nq):
    """kv_rows 0, k and v NULL: every row sees nothing and becomes zeros."""
    c = Call(45, nq, [0, 0], (20, 5), 64, "f16", tail=1)
    c.args.k = c.args.v = None
    c.args.kv_rows = 0
    c.run().check().free()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("m", [1, 33, 64, 129, 161, 4000])
def test_a_nan_in_a_key_that_a_row_sees_reaches_it_in_either_form(m, t):
    """The last key alone, the last 32 of a tile, and everything from the middle on: keys of which a wavefront, or a split, may hold
    nothing else.  max_q chooses the form; the other heads of the same token stay as they are."""
    for first in sorted({m - 1, (m - 1) // 32 * 32, m // 2, 0}):
        def edit(c, q, k, v):
            k[first:m, 1, ::3] = np.nan

        for max_q in (1, 200):
            one(46, [1, 1], [m, 70], (20, 5), 128, t, edit=edit, max_q=max_q)


def test_one_workspace_of_the_largest_need_serves_batches_of_every_size():
    """64 sequences need no workspace and fewer do: the largest of all sizes' needs is asked for once and serves them all."""
    calls = [Call(50 + n, [1] * n, [600 - 5 * i for i in range(n)], (16, 8), 64, "f16", max_kv=4000) for n in (64, 40, 9, 3, 1)]
    needs = [sp.attention_workspace_bytes(c.args) for c in calls]
    assert needs[0] == 0 and max(needs) > 0
    ws = sp.DeviceBuffer(max(needs))
    for c in calls:
        print("batch", c.args.batch, flush=True)
        c.ws = sp.DeviceBuffer(16)
        sp.attention(c.args, ws, ws.nbytes)
        sp.device_sync()
        c.got = c.out.to_numpy(np.float16, c.before.shape)
        c.check().free()
    ws.free()


@pytest.mark.parametrize("nq,max_q,heads,dim,max_kv", [([1, 1, 1, 1, 1], 1, (20, 5), 128, 3000), ([40, 9, 130, 2, 33], 200, (4, 2), 64, 100), ([40, 9, 130, 2, 33], 130, (6, 2), 128, 3000)])
def test_arrays_that_lead_astray_write_nothing_beside_the_rows(nq, max_q, heads, dim, max_kv):
    """All three forms, `out` between guard rows: cache rows and lengths of some sequences that lead out of the buffers (the others are
    exact all the same), then starts of the queries that do (nothing beside `out` and the workspace is written)."""
    c = Call(60, nq, [900, 20, 2500, 300, 40], heads, dim, "f16", max_q=max_q, max_kv=max_kv, tail=3)
    hq, guard = heads[0], 512
    rows = np.full((c.total + 2 * guard, hq * dim), 0x5A5A, np.uint16)
    rows[guard:-guard] = c.before.view(np.uint16)
    big = sp.DeviceBuffer.from_numpy(rows)
    c.args.out = big.ptr.value + 2 * guard * hq * dim
    start, length = c.kv_start.copy(), c.kv_len.copy()
    start[0], start[3] = -5, 1 << 30
    length[0], length[2], length[3] = 1 << 30, -7, 1 << 30
    n = sp.attention_workspace_bytes(c.args)
    c.ws = sp.DeviceBuffer(n + 4096)

    def call():
        c.ws.fill(0xFF)
        sp.attention(c.args, c.ws, n)
        sp.device_sync()
        got = big.to_numpy(np.uint16, rows.shape)
        assert (got[:guard] == 0x5A5A).all() and (got[-guard:] == 0x5A5A).all()
        assert (c.ws.to_numpy(np.uint8, n + 4096)[n:] == 0xFF).all()
        return got[guard:-guard]

    c.bufs[4].upload(start), c.bufs[5].upload(length)
    got = call()
    assert (got[-3:] == c.before[-3:].view(np.uint16)).all()  # the rows behind the last sequence
    values = op.widen(got.view(np.float16), "f16")
    want = op.attention(c.q, c.k, c.v, c.q_start, c.kv_start, np.array([0, c.kv_len[1], 0, 0, c.kv_len[4]]), c.scale, "f16")
    for row in [*range(c.q_start[1], c.q_start[2]), *range(c.q_start[4], c.q_start[5])]:
        assert (np.abs(values[row].reshape(hq, dim) - want[row][0]) <= want[row][1]).all(), row
    for bad in ([0, 9, 3, 1 << 30, 5, 7], [0, 60, 1, 70, 2, c.total], [-(1 << 31), (1 << 31) - 1] * 3, [(1 << 31) - 1, -1, 0, 1 << 30, 2, c.total + 1], [c.total] * 3 + [0, c.total, 1 << 30]):
        c.bufs[3].upload(np.array(bad, np.int64).astype(np.int32))
        call()
    big.free()
    c.free()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("nq,nk,max_q,max_kv", [([1, 1, 1], [300, 0, 77], 1, 2000), ([5, 70, 2], [5, 70, 2], 70, 70), ([30, 40, 9], [30, 1400, 600], 60, 2000)])
def test_rows_before_the_first_sequence_and_strides_of_their_own(nq, nk, max_q, max_kv, packed):
    """Starts that do not begin at 0, every buffer with another row stride, out's a multiple of 4 only."""
    hq, hkv, dim, before = 6, 2, 64, 11
    nk = nq if packed else nk
    r = np.random.default_rng(70)
    first = (before + np.concatenate([[0], np.cumsum(nq)])).astype(np.int32)
    start = first[:-1].copy() if packed else (3 + np.concatenate([[0], np.cumsum(nk)[:-1]])).astype(np.int32)
    total, rows = int(first[-1]) + 2, int(max(start + nk)) + 1
    (q, q64), (k, k64), (v, v64), (out, _) = (op.narrow(r.standard_normal((n, h * dim + pad)), "bf16") for n, h, pad in ((total, hq, 8), (rows, hkv, 40), (rows, hkv, 0), (total, hq, 4)))
    bufs = [sp.DeviceBuffer.from_numpy(x) for x in (q, k, v, out, first, start, np.asarray(nk, np.int32))]
    a = sp.AttentionArgs(q=bufs[0], k=bufs[1], v=bufs[2], out=bufs[3], q_stride=hq * dim + 8, k_stride=hkv * dim + 40, v_stride=hkv * dim, out_stride=hq * dim + 4, kv_rows=rows, q_start=bufs[4],
                         kv_start=None if packed else bufs[5], kv_len=None if packed else bufs[6], batch=len(nq), total_q=total, max_q=max_q, max_kv=max_kv, q_heads=hq, kv_heads=hkv, head_dim=dim,
                         type=sp.X_BF16, scale=op.softmax_scale(dim))
    ws = sp.DeviceBuffer(sp.attention_workspace_bytes(a) + 16)
    ws.fill(0xFF)
    print("rows before", nq, nk, packed, flush=True)
    sp.attention(a, ws, ws.nbytes)
    sp.device_sync()
    got = bufs[3].to_numpy(np.uint16, out.shape)
    want = op.attention(q64[:, : hq * dim].reshape(total, hq, dim), k64[:, : hkv * dim].reshape(rows, hkv, dim), v64.reshape(rows, hkv, dim), first, start, nk, a.scale, "bf16")
    for row in range(total):
        if row not in want:
            assert (got[row] == out[row]).all(), row
            continue
        assert (got[row, hq * dim:] == out[row, hq * dim:]).all()
        assert (np.abs(op.widen(got[row, : hq * dim], "bf16").reshape(hq, dim) - want[row][0]) <= want[row][1]).all(), row
    for b in [ws] + bufs:
        b.free()
