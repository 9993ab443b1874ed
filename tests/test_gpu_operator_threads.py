"""GPU: the operators between a layer's projections called by several host threads at once, each with its own stream, buffers and
workspace, one adapter set among them: the results are those of calls made one at a time, bit for bit."""
import threading

import numpy as np
import pytest

import operators64 as op
import sptmm_amd as sp

pytestmark = pytest.mark.gpu

HQ, HKV, D, K = 6, 2, 128, 512
N = (HQ + 2 * HKV) * D


class Work:
    def __init__(self, seed, nq, nk, adapters):
        r = np.random.default_rng(seed)
        self.T, rows = sum(nq), sum(nk)
        first, at = np.concatenate([[0], np.cumsum(nq)]), np.concatenate([[0], np.cumsum(nk)])
        row = np.concatenate([np.arange(a + n - q, a + n) for a, n, q in zip(at, nk, nq)])
        self.adapters, self.stream = adapters, sp.Stream()
        dev = lambda x: sp.DeviceBuffer.from_numpy(np.ascontiguousarray(x))  # noqa: E731
        bits = lambda *s: op.narrow(r.standard_normal(s), "bf16")[0]  # noqa: E731
        self.bufs = dict(x=dev(bits(self.T, K)), base=dev(r.standard_normal((self.T, N)).astype(np.float32)), y=sp.DeviceBuffer(4 * self.T * N), q=sp.DeviceBuffer(2 * self.T * HQ * D),
                         slot=dev(r.integers(-1, 3, self.T).astype(np.int32)), k=dev(bits(rows, HKV * D)), v=dev(bits(rows, HKV * D)), row=dev(row.astype(np.int32)),
                         first=dev(first.astype(np.int32)), start=dev(at[:-1].astype(np.int32)), n=dev(np.array(nk, np.int32)), out=sp.DeviceBuffer(2 * self.T * HQ * D))
        b = self.bufs
        y = b["y"].ptr.value
        self.heads = sp.HeadsArgs(q=y, k=y + 4 * HQ * D, v=y + 4 * (HQ + HKV) * D, q_stride=N, k_stride=N, v_stride=N, in_type=sp.X_F32, out_type=sp.X_BF16, q_out=b["q"], k_out=b["k"],
                                  v_out=b["v"], q_out_stride=HQ * D, k_out_stride=HKV * D, v_out_stride=HKV * D, tokens=self.T, q_heads=HQ, kv_heads=HKV, head_dim=D, positions=b["row"],
                                  kv_rows=b["row"], kv_capacity=rows, rotation=sp.Rotation(op.frequencies(D)))
        self.attn = sp.AttentionArgs(q=b["q"], k=b["k"], v=b["v"], out=b["out"], q_stride=HQ * D, k_stride=HKV * D, v_stride=HKV * D, out_stride=HQ * D, kv_rows=rows, q_start=b["first"],
                                     kv_start=b["start"], kv_len=b["n"], batch=len(nq), total_q=self.T, max_q=max(nq), max_kv=max(nk), q_heads=HQ, kv_heads=HKV, head_dim=D, type=sp.X_BF16,
                                     scale=op.softmax_scale(D))
        self.ws = sp.DeviceBuffer(max(256, sp.attention_workspace_bytes(self.attn), adapters.workspace_bytes(self.T)))

    def run(self):
        b, st, n = self.bufs, self.stream, self.ws.nbytes
        self.adapters.apply(b["x"], b["slot"], self.T, b["base"], b["y"], self.ws, n, st)
        sp.heads_norm_rotate(self.heads, st)
        sp.attention(self.attn, self.ws, n, st)
        st.sync()
        return b["out"].to_numpy(np.uint16, (self.T, HQ * D)), b["y"].to_numpy(np.uint32, (self.T, N))

    def free(self):
        for b in [*self.bufs.values(), self.ws]:
            b.free()
        self.stream.destroy()


def test_threads_at_once():
    sp.device_init(0)
    r = np.random.default_rng(1)
    a = sp.Adapters(K, N, sp.X_BF16, 3, 40)
    for slot, rank in enumerate((16, 40, 3)):
        A, B = (sp.DeviceBuffer.from_numpy(op.narrow(r.standard_normal(s) * 0.1, "bf16")[0]) for s in ((rank, K), (N, rank)))
        a.set(slot, A, B, rank, 0.5)
        sp.device_sync()
        A.free(), B.free()
    work = [Work(2, [1] * 9, [1, 700, 3, 5000, 40, 2, 33, 1500, 9], a), Work(3, [70, 120], [3000, 1200], a), Work(4, [300, 1, 57], [300, 1, 57], a), Work(5, [1], [4000], a)]
    alone = [w.run() for w in work]
    wrong = []

    def worker(i):
        try:
            for rep in range(12):
                if not all((x == y).all() for x, y in zip(work[i].run(), alone[i])):
                    wrong.append((i, rep))
        except Exception as e:  # (an exception in a thread would pass silently)
            wrong.append((i, e))

    print("threads: 4 x 12 rounds", flush=True)
    threads = [threading.Thread(target=worker, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    for w in work:
        w.free()
    a.free()
