"""GPU: low-rank adapters beside a projection (sptmm_adapters_*) against the definition in 64 bits."""
import numpy as np
import pytest

import operators64 as op
import sptmm_amd as sp

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    return sp.device_init(0)


class Set:
    def __init__(self, seed, K, N, t, ranks, max_rank=None):
        r = np.random.default_rng(seed)
        self.K, self.N, self.t = K, N, t
        self.a = sp.Adapters(K, N, op.CODE[t], len(ranks), max_rank or max(ranks))
        self.A, self.B, self.scale = [], [], []
        for i, k in enumerate(ranks):
            self.put(i, r, k, append=True)

    def put(self, slot, r, k, append=False, edit=None):
        A, B = r.standard_normal((k, self.K)) / np.sqrt(self.K), r.standard_normal((self.N, k))
        if edit:
            edit(A, B)
        (ab, a64), (bb, b64) = op.narrow(A, self.t), op.narrow(B, self.t)
        scale = float(np.float32(r.uniform(0.25, 2.0)))
        bufs = [sp.DeviceBuffer.from_numpy(x) if x.size else sp.DeviceBuffer(16) for x in (ab, bb)]
        self.a.set(slot, bufs[0], bufs[1], k, scale)
        sp.device_sync()
        for b in bufs:
            b.free()
        for lst, x in ((self.A, a64), (self.B, b64), (self.scale, scale)):
            lst.append(x) if append else lst.__setitem__(slot, x)

    def check(self, seed, slot, base="other", edit=None):
        r = np.random.default_rng(seed)
        M, slot = len(slot), np.asarray(slot, np.int32)
        x = r.standard_normal((M, self.K))
        if edit:
            edit(x)
        xb, x64 = op.narrow(x, self.t)
        b32 = r.standard_normal((M, self.N)).astype(np.float32)
        n = self.a.workspace_bytes(M)
        X, S, base_buf = sp.DeviceBuffer.from_numpy(xb), sp.DeviceBuffer.from_numpy(slot), sp.DeviceBuffer.from_numpy(b32)
        Y, ws = sp.DeviceBuffer(4 * M * self.N + 64), sp.DeviceBuffer(n + 256)
        Y.fill(0xFF)
        ws.fill(0xFF)
        print("adapters M", M, "K", self.K, "N", self.N, self.t, "base", base, flush=True)
        if base == "in place":
            self.a.apply(X, S, M, base_buf, base_buf, ws, n)
        else:
            self.a.apply(X, S, M, None if base == "none" else base_buf, Y, ws, n)
        sp.device_sync()
        assert (ws.to_numpy(np.uint8, n + 256)[n:] == 0xFF).all()
        assert (Y.to_numpy(np.uint8, 4 * M * self.N + 64)[4 * M * self.N:] == 0xFF).all()
        got = (base_buf if base == "in place" else Y).to_numpy(np.float32, (M, self.N)).astype(np.float64)
        with np.errstate(invalid="ignore"):
            want, bound = op.adapters(x64, slot, np.zeros((M, self.N)) if base == "none" else b32.astype(np.float64), self.A, self.B, self.scale)
        fine = np.isfinite(want)
        bad = np.argwhere(np.isnan(got) != np.isnan(want))
        assert not len(bad), (len(bad), bad[:3], got[tuple(bad[0])], want[tuple(bad[0])], slot[bad[0][0]])
        assert (got[~fine & ~np.isnan(want)] == want[~fine & ~np.isnan(want)]).all()
        off = np.abs(got - want)
        assert (off[fine] <= bound[fine]).all(), float((off[fine] / bound[fine]).max())
        for o in (X, S, base_buf, Y, ws):
            o.free()
        return got

    def free(self):
        self.a.free()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("K,N", [(16, 16), (48, 32), (272, 80), (2560, 640), (6912, 144)])
def test_shapes_and_ranks(K, N, t):
    s = Set(1, K, N, t, [1, 8, 16, 17, 33, 64, 3])
    r = np.random.default_rng(2)
    for M in (1, 2, 15, 16, 17, 40, 130, 300):
        s.check(M, r.integers(-1, 8, M))  # 7 and -1: no adapter
    s.free()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("K,N,rank", [(2560, 3840, 16), (2576, 272, 9), (1024, 528, 75)])
def test_a_few_rows(K, N, rank, t):
    s = Set(10, K, N, t, [rank, 1, rank, 3, rank])
    for M in (1, 2, 7, 16):
        s.check(M, (np.arange(M) * 3 + 2) % 6 - 1)
        s.check(M + 50, np.full(M, 2), "in place")
    assert s.a.workspace_bytes(1) == 0  # small weights: both products in one launch
    s.free()


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_many_rows(t):
    """Enough rows and columns for the second product on the 16-bit matrix instruction, by parts of h."""
    s = Set(11, 48, 2064, t, [1, 16, 40, 7, 64])
    r = np.random.default_rng(1)
    M = 2100
    s.check(1, np.sort(r.integers(-1, 6, M)))
    s.check(2, r.integers(-1, 6, M), "in place")

    def spread(x):  # sums of very different size, and rows that are not finite
        x[::3] *= 1e4 if t == "f16" else 1e20
        x[1::3] *= 1e-4 if t == "f16" else 1e-20
        x[2, 3], x[900, 0], x[1500, 7] = np.inf, np.nan, -np.inf
        x[40] = 0.0
    s.check(3, np.arange(M) // 40 % 6, edit=spread)
    s.put(1, r, 16, edit=lambda A, B: B.__setitem__((70, 3), np.inf))
    s.check(4, np.arange(M) // 9 % 6 - 1)
    s.free()


@pytest.mark.parametrize("M,K,N,rank", [(4, 2560, 384, 64), (1, 2560, 13824, 64), (2, 2592, 256, 64), (16, 2560, 13824, 16), (5, 2560, 13824, 16), (12, 6912, 2560, 16)])
def test_sides_of_the_single_launch(M, K, N, rank):
    """320 KiB of A a slot and more, and reads of A by all workgroups of 32 MiB and more."""
    s = Set(13, K, N, "f16", [rank] * 17, rank)
    s.check(1, np.arange(M) % 17)
    s.free()


@pytest.mark.parametrize("M", [512, 516, 390])
def test_sides_of_the_many_row_form(M):
    s = Set(14, 64, 6912, "bf16", [8, 0, 40, 64, 17], 64)  # 54 workgroups of columns to every 64 rows
    s.check(1, np.arange(M) * 7 % 6 - 1)
    s.free()


def test_many_rows_of_the_largest_rank():
    s = Set(12, 32, 2064, "bf16", [256, 3, 250], 256)
    s.check(1, np.arange(2100) // 30 % 4 - 1)
    s.free()


@pytest.mark.parametrize("rank,max_rank", [(1, 256), (64, 64), (65, 128), (200, 256), (256, 256)])
def test_large_ranks(rank, max_rank):
    s = Set(3, 320, 96, "bf16", [rank, 5], max_rank)
    for M in (1, 20, 200):
        s.check(M, np.arange(M) % 3 - 1)
    s.free()


@pytest.mark.parametrize("base", ["other", "in place", "none"])
@pytest.mark.parametrize("M", [1, 9, 48, 150])
def test_base_in_place_and_none(M, base):
    s = Set(4, 512, 256, "f16", [16, 4, 40])
    s.check(5, np.random.default_rng(M).integers(-1, 3, M), base)
    s.free()


@pytest.mark.parametrize("M", [16, 64, 129, 400])
def test_one_slot_for_all_every_row_another_and_runs(M):
    ranks = [int(x) for x in np.random.default_rng(1).integers(1, 30, 64)]
    s = Set(5, 256, 128, "bf16", ranks)
    s.check(1, np.zeros(M))
    s.check(2, np.arange(M) % 64)
    s.check(3, np.arange(M) // 7 % 64)
    s.check(4, np.full(M, -1))
    s.check(5, np.where(np.arange(M) % 2, 1 << 30, -(1 << 31)))  # far out of range: no adapter
    s.free()


def test_slots_are_replaced_and_emptied():
    s = Set(6, 128, 64, "f16", [8, 8, 8], 40)
    r = np.random.default_rng(9)
    slot = np.arange(30) % 3
    s.check(1, slot)
    s.put(1, r, 40)
    s.check(2, slot)
    s.put(1, r, 2)
    s.check(3, slot)
    s.put(1, r, 0)
    got = s.check(4, slot)
    assert np.isfinite(got).all()
    s.free()


@pytest.mark.parametrize("M", [17, 200])
@pytest.mark.parametrize("what", [np.inf, np.nan])
def test_what_is_not_finite_reaches_its_own_rows_only(what, M):
    s = Set(7, 128, 64, "bf16", [8, 20, 8])
    r = np.random.default_rng(3)

    def in_b(A, B):
        B[5, 3] = what

    def in_a(A, B):
        A[2, 7] = what
    s.put(1, r, 20, edit=in_b)
    s.put(2, r, 8, edit=in_a)
    got = s.check(1, np.arange(M) % 4 - 1)
    assert np.isfinite(got[np.arange(M) % 4 < 2]).all()

    def row(x):
        x[3, 11] = what
    s.check(2, np.arange(M) % 2 - 1, edit=row)
    s.free()


def test_a_captured_call_follows_its_buffers():
    K, N, M = 512, 320, 33
    s = Set(8, K, N, "bf16", [16, 9, 30])
    st = sp.Stream()
    n = s.a.workspace_bytes(M)
    X, S, base, Y, Z, ws = (sp.DeviceBuffer(x) for x in (2 * M * K, 4 * M, 4 * M * N, 4 * M * N, 4 * M * N, n))
    S.upload(np.zeros(M, np.int32))
    with sp.Graph(st) as g:
        s.a.apply(X, S, M, base, Y, ws, n, st)
    r = np.random.default_rng(5)
    for rep in range(3):
        print("replay", rep, flush=True)
        xb, x64 = op.narrow(r.standard_normal((M, K)), "bf16")
        b32, slot = r.standard_normal((M, N)).astype(np.float32), r.integers(-1, 3, M).astype(np.int32)
        X.upload(xb), S.upload(slot), base.upload(b32)
        g.launch(st)
        st.sync()
        got = Y.to_numpy(np.float32, (M, N))
        want, bound = op.adapters(x64, slot, b32.astype(np.float64), s.A, s.B, s.scale)
        assert (np.abs(got - want) <= bound).all()
        s.a.apply(X, S, M, base, Z, ws, n, st)
        st.sync()
        assert (Z.to_numpy(np.float32, (M, N)) == got).all()
    g.destroy()
    for o in (X, S, base, Y, Z, ws, s):
        o.free()
    st.destroy()


def test_refusals():
    s = Set(9, 6912, 32, "f16", [4, 4], 64)
    n = s.a.workspace_bytes(3)
    assert n > 0 and s.a.workspace_bytes(0) == 0 and s.a.workspace_bytes(-3) == 0
    X, S, Y, ws = sp.DeviceBuffer(2 * 3 * 6912 + 16), sp.DeviceBuffer(16), sp.DeviceBuffer(4 * 3 * 32 + 16), sp.DeviceBuffer(n + 16)
    off = X.ptr.value + 2
    for a in ((None, S, 3, None, Y, ws, n), (X, None, 3, None, Y, ws, n), (X, S, 3, None, None, ws, n), (X, S, 3, None, Y, None, n), (X, S, 0, None, Y, ws, n), (X, S, -1, None, Y, ws, n),
              (X, S, 3, None, Y, ws, n - 1), (X, S, (1 << 24) + 1, None, Y, ws, n), (off, S, 3, None, Y, ws, n), (X, S.ptr.value + 2, 3, None, Y, ws, n), (X, S, 3, Y.ptr.value + 4, Y, ws, n)):
        with pytest.raises(sp.SptmmError):
            s.a.apply(*a)
    with pytest.raises(sp.SptmmError) as e:  # more tiles than a launch has work-items
        Set(1, 16, 1 << 14, "f16", [1]).a.apply(X, S, 1 << 24, None, Y, ws, 1 << 60)
    assert e.value.code == -2
    for a in ((-1, X, Y, 4, 1.0), (2, X, Y, 4, 1.0), (0, X, Y, 65, 1.0), (0, X, Y, -1, 1.0), (0, None, Y, 4, 1.0), (0, X, None, 4, 1.0), (0, X, Y, 4, float("nan")), (0, X, Y, 4, float("inf"))):
        with pytest.raises(sp.SptmmError):
            s.a.set(*a)
    s.check(1, [0, 1, 0])
    for o in (X, S, Y, ws, s):
        o.free()


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_a_small_inner_sum_beside_a_large_one_keeps_its_bits(t):
    """Rank 0's inner sum is some 2^28 times rank 1's, and the even columns do not use it: what they add is rank 1's alone."""
    s = Set(15, 48, 2064, t, [2, 3])

    def edit(A, B):
        A[0] *= 6e4
        A[1] *= 2e-4
        B[::2, 0] = 0.0

    s.put(0, np.random.default_rng(1), 2, edit=edit)
    for M in (5, 100, 2100):  # all three forms
        s.check(2, np.arange(M) // 40 % 3 - 1, "none")
    s.free()


@pytest.mark.parametrize("rank", [192, 193, 256])
def test_many_rows_of_large_ranks_in_fp16(rank):
    s = Set(19, 32, 2064, "f16", [rank, 3, rank - 5], rank)
    s.check(1, np.arange(2100) // 30 % 4 - 1)
    s.free()


def test_a_captured_set_of_weights_is_what_its_buffers_hold():
    """Replays of one captured set: with a B that is not finite, then with an ordinary one.  The second gives, bit for bit, what a
    set that never held anything else gives."""
    K, N, M, rank = 48, 2064, 2100, 16
    st = sp.Stream()
    r = np.random.default_rng(16)
    (ab, a64), (bb, b64), (xb, x64) = (op.narrow(r.standard_normal(n), "bf16") for n in ((rank, K), (N, rank), (M, K)))
    wild = bb.copy()
    wild[70, 3] = 0x7F80  # infinity
    A, B, X, S = (sp.DeviceBuffer.from_numpy(v) for v in (ab, wild, xb, np.zeros(M, np.int32)))
    one, other = sp.Adapters(K, N, sp.X_BF16, 2, rank), sp.Adapters(K, N, sp.X_BF16, 2, rank)
    n = one.workspace_bytes(M)
    ws, Y, Z = sp.DeviceBuffer(n), sp.DeviceBuffer(4 * M * N), sp.DeviceBuffer(4 * M * N)
    with sp.Graph(st) as g:
        one.set(0, A, B, rank, 0.5, st)
        one.apply(X, S, M, None, Y, ws, n, st)
    for rep, b in enumerate((wild, bb, wild, bb)):
        print("replay", rep, flush=True)
        B.upload(b)
        g.launch(st)
        other.set(rep % 2, A, B, rank, 0.5, st)
        S.upload(np.full(M, 0, np.int32))
        st.sync()
        got = Y.to_numpy(np.float32, (M, N))
        with np.errstate(invalid="ignore"):
            want, bound = op.adapters(x64, np.zeros(M, int), np.zeros((M, N)), [a64], [op.widen(b, "bf16")], [0.5])
        fine = np.isfinite(want)
        assert (np.isfinite(got) == fine).all() and (np.abs(got - want)[fine] <= bound[fine]).all()
        fresh = sp.Adapters(K, N, sp.X_BF16, 2, rank)
        fresh.set(0, A, B, rank, 0.5, st)
        fresh.apply(X, S, M, None, Z, ws, n, st)
        st.sync()
        assert (Z.to_numpy(np.uint32, (M, N)) == got.view(np.uint32)).all(), rep
        fresh.free()
    g.destroy()
    for o in (A, B, X, S, ws, Y, Z, one, other):
        o.free()
    st.destroy()


def test_a_refused_allocation_leaves_no_error_behind():
    """35 TB of weights: refused.  The call after it, on the same thread, is not blamed for it."""
    s = Set(17, 64, 64, "f16", [4, 2])
    with pytest.raises(sp.SptmmError) as e:
        sp.Adapters(1 << 20, 1 << 20, sp.X_F16, 65536, 256)
    assert e.value.code == -4 and "memory" in str(e.value)
    s.check(1, [0, 1, -1])
    with pytest.raises(sp.SptmmError):
        sp.DeviceBuffer(1 << 50)
    X, slot, Y = sp.DeviceBuffer(2 * 64), sp.DeviceBuffer.from_numpy(np.zeros(1, np.int32)), sp.DeviceBuffer(4 * 64)
    X.fill(0)
    with pytest.raises(sp.SptmmError):
        sp.DeviceBuffer(1 << 50)
    s.a.apply(X, slot, 1, None, Y, None, 0)
    sp.device_sync()
    for o in (X, slot, Y, s):
        o.free()


def test_one_workspace_for_the_largest_call_serves_the_smaller_ones():
    s = Set(18, 2560, 64, "f16", [16, 3])
    sizes = [4096, 4095, 4081, 4080, 2049, 1024, 1008, 500, 257, 130, 129, 128, 113, 112, 49, 48, 17, 16, 15, 2, 1]
    n = s.a.workspace_bytes(4096)
    assert all(s.a.workspace_bytes(a) >= s.a.workspace_bytes(b) for a, b in zip(sizes, sizes[1:]))
    (xb, x64), slot = op.narrow(np.random.default_rng(1).standard_normal((4096, 2560)), "f16"), (np.arange(4096) % 3 - 1).astype(np.int32)
    want, bound = op.adapters(x64, slot, np.zeros((4096, 64)), s.A, s.B, s.scale)
    ws, X, Y, S = sp.DeviceBuffer(n), sp.DeviceBuffer.from_numpy(xb), sp.DeviceBuffer(4 * 4096 * 64), sp.DeviceBuffer.from_numpy(slot)
    for M in sizes:
        print("M", M, flush=True)
        s.a.apply(X, S, M, None, Y, ws, n)
        sp.device_sync()
        assert (np.abs(Y.to_numpy(np.float32, (M, 64)) - want[:M]) <= bound[:M]).all()
    for o in (ws, X, Y, S, s):
        o.free()
