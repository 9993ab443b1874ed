"""GPU: norms of query and key heads with the rotation in the same pass (sptmm_heads_norm_rotate) against the definition in 64 bits."""
import numpy as np
import pytest

import operators64 as op
import sptmm_amd as sp

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    return sp.device_init(0)


def run(seed, T, hq, hkv, D, tin="f32", tout="bf16", rotated=None, interleaved=False, gains="qk", pad=0, shift=0, far=5000, rows="scatter", values=True, eps=1e-5, edit=None, freq=None):
    """One call on a fused row [q | k | v] (plus `pad` elements, starting `shift` elements into the buffer), checked."""
    print("heads", T, hq, hkv, D, tin, tout, rotated, interleaved, gains, pad, shift, rows, flush=True)
    r = np.random.default_rng(seed)
    H = hq + 2 * hkv
    x = r.standard_normal((T, H * D + pad)) * 2.0
    if edit:
        edit(x)
    host, x64 = op.narrow(x, tin)
    flat = np.zeros(host.size + shift, host.dtype)
    flat[shift:] = host.ravel()
    src = sp.DeviceBuffer.from_numpy(flat)
    esz = host.itemsize
    at = src.ptr.value + shift * esz
    pos = r.integers(-far, far, T).astype(np.int32)
    cap = T + 5
    row = np.arange(T, dtype=np.int32) if rows is None else r.permutation(cap)[:T].astype(np.int32)
    if rows == "some":
        row[::3] = np.where(np.arange(len(row[::3])) % 2, cap, -7)  # padding: not stored
    gq, gk = (1 + 0.3 * r.standard_normal(D)).astype(np.float32), (1 + 0.3 * r.standard_normal(D)).astype(np.float32)
    freq = op.frequencies(D if rotated is None else rotated) if freq is None else freq
    dt = op.buffer_type(tout)
    outs, before = [], []
    for n, rr in ((hq, T), (hkv, cap), (hkv, cap)):
        b, _ = op.narrow(r.standard_normal((rr, n * D + pad)), tout)
        before.append(b)
        outs.append(sp.DeviceBuffer.from_numpy(b) if b.size else sp.DeviceBuffer(16))
    small = [sp.DeviceBuffer.from_numpy(v) for v in (pos, row, gq, gk)]
    a = sp.HeadsArgs(q=at, k=at + hq * D * esz, v=at + (hq + hkv) * D * esz if values else None, q_stride=H * D + pad, k_stride=H * D + pad, v_stride=H * D + pad, in_type=op.CODE[tin],
                     out_type=op.CODE[tout], q_out=outs[0], k_out=outs[1], v_out=outs[2], q_out_stride=hq * D + pad, k_out_stride=hkv * D + pad, v_out_stride=hkv * D + pad,
                     tokens=T, q_heads=hq, kv_heads=hkv, head_dim=D, positions=small[0], kv_rows=None if rows is None else small[1], kv_capacity=cap,
                     q_gain=small[2] if "q" in gains else None, k_gain=small[3] if "k" in gains else None, eps=eps, rotation=sp.Rotation(freq, interleaved) if len(freq) else None)
    sp.heads_norm_rotate(a)
    sp.device_sync()
    got = [o.to_numpy(dt, b.shape) for o, b in zip(outs, before)]
    heads = x64[:, : H * D].reshape(T, H, D)
    with np.errstate(invalid="ignore"):
        want = [op.rotate_norm(heads[:, :hq], pos, gq if "q" in gains else None, eps, freq, interleaved, tout),
                op.rotate_norm(heads[:, hq:hq + hkv], pos, gk if "k" in gains else None, eps, freq, interleaved, tout),
                (heads[:, hq + hkv:], np.abs(heads[:, hq + hkv:]) * op.HALF_STEP[tout] + op.TINY[tout])]
    for i, (n, rr) in enumerate(((hq, T), (hkv, cap), (hkv, cap))):
        touched = np.zeros(before[i].shape, bool)
        for t in range(T):
            at_row = t if i == 0 else int(row[t])
            if not 0 <= at_row < rr or (i == 2 and not values):
                continue
            touched[at_row, : n * D] = True
            w, e = want[i][0][t].ravel(), want[i][1][t].ravel()
            g = op.widen(got[i][at_row, : n * D], tout)
            fine = np.isfinite(w)
            assert (np.isnan(g) == np.isnan(w)).all(), ("NaN", i, t)
            off = np.abs(g - w)[fine]
            assert (off <= e[fine]).all(), (i, t, float((off / e[fine]).max()))
        same = got[i].view(np.uint16) == before[i].view(np.uint16)
        assert same[~touched].all(), "something was written outside the rows"
    for o in [src] + outs + small:
        o.free()
    return got


@pytest.mark.parametrize("tin", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tout", ["f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types_and_pairings(tin, tout, interleaved):
    run(1, 37, 20, 5, 128, tin, tout, interleaved=interleaved)
    run(2, 9, 4, 2, 64, tin, tout, rotated=24, interleaved=interleaved, rows="some")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D", [2, 6, 8, 16, 32, 34, 80, 96, 100, 128, 250, 256])
def test_widths(D, interleaved):
    run(3, 11, 3, 2, D, interleaved=interleaved)
    run(4, 5, 3, 1, D, "f16", "f16", rotated=D // 2 // 2 * 2, interleaved=interleaved)


@pytest.mark.parametrize("T", [1, 2, 3, 64, 2047, 2048, 2051])
def test_token_counts(T):
    run(5, T, 4, 1, 64, "bf16", "bf16")


@pytest.mark.parametrize("gains", ["", "q", "k", "qk"])
def test_norms_of_either_kind_of_head(gains):
    run(6, 10, 4, 2, 64, gains=gains)
    run(7, 10, 4, 2, 64, gains=gains, freq=[])


def test_head_counts_and_missing_parts():
    run(8, 6, 5, 0, 64)
    run(9, 6, 0, 3, 64)
    run(10, 6, 2, 3, 64, values=False)
    run(11, 6, 33, 7, 32, rows=None)


@pytest.mark.parametrize("shift,pad", [(0, 4), (4, 0), (1, 0), (2, 3), (0, 1)])
def test_alignment_and_strides(shift, pad):
    for tin in ("f32", "f16"):
        run(12, 8, 4, 2, 64, tin, "f16", shift=shift, pad=pad)
        run(13, 8, 4, 2, 64, tin, "bf16", shift=shift, pad=pad, interleaved=True)


def test_far_positions():
    run(14, 64, 2, 1, 128, far=2 ** 31 - 1)
    run(15, 64, 2, 1, 64, far=2 ** 30, freq=[1.0, 0.5, 3.0, 1e-6, 6.283185307179586, 100.25, -0.75, 0.0])


def test_rows_of_zeros_and_what_is_not_finite():
    def zeros(x):
        x[2] = 0.0
    run(16, 5, 2, 1, 64, edit=zeros, eps=1e-5)

    def bad(x):
        x[1, 3] = np.nan
        x[2, 70] = np.nan
        x[3, 140] = np.nan
    got = run(17, 6, 1, 1, 64, edit=bad, rows=None)
    assert np.isnan(op.widen(got[0][1], "bf16")).all() and not np.isnan(op.widen(got[0][2], "bf16")).any()


def test_written_over_its_own_input():
    """16-bit rows, the outputs being the inputs."""
    T, hq, hkv, D = 50, 4, 2, 64
    r = np.random.default_rng(4)
    host, x64 = op.narrow(r.standard_normal((T, (hq + 2 * hkv) * D)), "f16")
    buf = sp.DeviceBuffer.from_numpy(host)
    p = buf.ptr.value
    S, q, k, v = (hq + 2 * hkv) * D, p, p + 2 * hq * D, p + 2 * (hq + hkv) * D
    gain = np.ones(D, np.float32)
    g = sp.DeviceBuffer.from_numpy(gain)
    freq = op.frequencies(D)
    a = sp.HeadsArgs(q=q, k=k, v=v, q_stride=S, k_stride=S, v_stride=S, in_type=1, out_type=1, q_out=q, k_out=k, v_out=v, q_out_stride=S, k_out_stride=S, v_out_stride=S, tokens=T,
                     q_heads=hq, kv_heads=hkv, head_dim=D, kv_capacity=T, q_gain=g, k_gain=g, eps=1e-6, rotation=sp.Rotation(freq))
    sp.heads_norm_rotate(a)
    sp.device_sync()
    got = op.widen(buf.to_numpy(np.float16, host.shape), "f16").reshape(T, -1, D)
    w, e = op.rotate_norm(x64.reshape(T, -1, D)[:, : hq + hkv], np.arange(T), gain.astype(np.float64), 1e-6, freq, False, "f16")  # positions NULL: 0, 1, 2, ...
    assert (np.abs(got[:, : hq + hkv] - w) <= e).all()
    assert (got[:, hq + hkv:] == x64.reshape(T, -1, D)[:, hq + hkv:]).all()
    buf.free()
    g.free()
