"""GPU: the attention half of a decoder layer run through the library as a program runs it, on one stream and as a replayed graph:

    q+k+v projection (quantised rows, ternary weights) -> adapters -> heads (norms, rotation, cache) -> attention -> o projection -> adapters

a prompt of several sequences first, then single tokens against the caches it left.  Every stage is checked against its definition in
64 bits on the bits that the stage before left on the device, so that no stage's rounding hides another's fault."""
import numpy as np
import pytest

import operators64 as op
import oracle
import sptmm_amd as sp

pytestmark = pytest.mark.gpu

K, HQ, HKV, D = 512, 4, 2, 64
NQKV, NQ = (HQ + 2 * HKV) * D, HQ * D
T16 = "bf16"
CAP = 200  # cache rows per sequence


class Block:
    def __init__(self, seed):
        r = np.random.default_rng(seed)
        self.w_qkv = sp.generate_ternary_iid(K, NQKV, 5, 0.3, 0.3)
        self.w_o = sp.generate_ternary_iid(NQ, K, 6, 0.3, 0.3)
        self.qkv, self.o = sp.Weights.upload_dense(self.w_qkv, sp.KIND_U16, 32), sp.Weights.upload_dense(self.w_o, sp.KIND_DELTA, 32)
        self.sets, self.lora = [], []
        for k, n in ((K, NQKV), (NQ, K)):
            a = sp.Adapters(k, n, op.CODE[T16], 3, 16)
            host = ([], [], [])
            for slot, rank in enumerate((16, 5, 9)):
                (ab, a64), (bb, b64) = op.narrow(r.standard_normal((rank, k)) / np.sqrt(k), T16), op.narrow(r.standard_normal((n, rank)) * 0.5, T16)
                da, db = sp.DeviceBuffer.from_numpy(ab), sp.DeviceBuffer.from_numpy(bb)
                a.set(slot, da, db, rank, 0.5)
                sp.device_sync()
                da.free(), db.free()
                for h, x in zip(host, (a64, b64, 0.5)):
                    h.append(x)
            self.sets.append(a)
            self.lora.append(host)
        self.gains = [(1 + 0.2 * r.standard_normal(D)).astype(np.float32) for _ in range(2)]
        self.gain_bufs = [sp.DeviceBuffer.from_numpy(g) for g in self.gains]
        self.freq = op.frequencies(D)
        self.rotation = sp.Rotation(self.freq)

    def buffers(self, T, batch, max_q, max_kv):
        b = {n: sp.DeviceBuffer(x) for n, x in (("x", 2 * T * K), ("slot", 4 * T), ("y", 4 * T * NQKV), ("y1", 4 * T * NQKV), ("pos", 4 * T), ("row", 4 * T), ("q", 2 * T * NQ),
                                                ("first", 4 * (batch + 1)), ("start", 4 * batch), ("len", 4 * batch), ("att", 2 * T * NQ), ("z", 4 * T * K), ("z1", 4 * T * K))}
        b["heads"] = sp.HeadsArgs(q=b["y1"], k=b["y1"].ptr.value + 4 * NQ, v=b["y1"].ptr.value + 4 * (NQ + HKV * D), q_stride=NQKV, k_stride=NQKV, v_stride=NQKV, in_type=sp.X_F32,
                                  out_type=op.CODE[T16], q_out=b["q"], k_out=self.k, v_out=self.v, q_out_stride=NQ, k_out_stride=HKV * D, v_out_stride=HKV * D, tokens=T, q_heads=HQ,
                                  kv_heads=HKV, head_dim=D, positions=b["pos"], kv_rows=b["row"], kv_capacity=self.rows, q_gain=self.gain_bufs[0], k_gain=self.gain_bufs[1], eps=1e-5,
                                  rotation=self.rotation)
        b["attn"] = sp.AttentionArgs(q=b["q"], k=self.k, v=self.v, out=b["att"], q_stride=NQ, k_stride=HKV * D, v_stride=HKV * D, out_stride=NQ, kv_rows=self.rows, q_start=b["first"],
                                     kv_start=b["start"], kv_len=b["len"], batch=batch, total_q=T, max_q=max_q, max_kv=max_kv, q_heads=HQ, kv_heads=HKV, head_dim=D, type=op.CODE[T16],
                                     scale=op.softmax_scale(D))
        b["n"] = max(16, sp.attention_workspace_bytes(b["attn"]), *(s.workspace_bytes(T) for s in self.sets), self.qkv.q8_workspace_bytes(T), self.o.q8_workspace_bytes(T))
        b["ws"] = sp.DeviceBuffer(b["n"])
        return b

    def issue(self, b, T, st):
        self.qkv.gemv_q8_ws(b["x"], 2, T, 0.04, b["y"], b["ws"], b["n"], st)
        self.sets[0].apply(b["x"], b["slot"], T, b["y"], b["y1"], b["ws"], b["n"], st)
        sp.heads_norm_rotate(b["heads"], st)
        sp.attention(b["attn"], b["ws"], b["n"], st)
        self.o.gemv_q8_ws(b["att"], 2, T, 0.05, b["z"], b["ws"], b["n"], st)
        self.sets[1].apply(b["att"], b["slot"], T, b["z"], b["z1"], b["ws"], b["n"], st)

    def check(self, b, T, x64, slot, pos, row, first, start, length, before):
        y = b["y"].to_numpy(np.float32, (T, NQKV))
        quant, a = oracle.quantise_rows(x64.astype(np.float32))
        assert (y == oracle.rescale(oracle.dense_i8(quant, self.w_qkv), a, 0.04)).all()
        y1 = b["y1"].to_numpy(np.float32, (T, NQKV))
        want, e = op.adapters(x64, slot, y.astype(np.float64), *self.lora[0])
        assert (np.abs(y1 - want) <= e).all()
        heads = y1.astype(np.float64).reshape(T, -1, D)
        q = op.widen(b["q"].to_numpy(np.uint16, (T, HQ, D)), T16)
        kc, vc = (op.widen(c.to_numpy(np.uint16, (self.rows, HKV, D)), T16) for c in (self.k, self.v))
        for got, part, gain in ((q, heads[:, :HQ], self.gains[0]), (kc[row], heads[:, HQ:HQ + HKV], self.gains[1])):
            w, e = op.rotate_norm(part, pos, gain.astype(np.float64), 1e-5, self.freq, False, T16)
            assert (np.abs(got - w) <= e).all()
        assert (np.abs(vc[row] - heads[:, HQ + HKV:]) <= np.abs(heads[:, HQ + HKV:]) * op.HALF_STEP[T16] + op.TINY[T16]).all()
        old = np.ones(self.rows, bool)
        old[row] = False
        assert (kc[old] == before[0][old]).all() and (vc[old] == before[1][old]).all()  # the caches' other rows are as they were
        att_bits = b["att"].to_numpy(np.uint16, (T, NQ))
        att = op.widen(att_bits, T16)
        want = op.attention(q, kc, vc, first, start, length, op.softmax_scale(D), T16)
        for t in range(T):
            o, e = want[t]
            assert (np.abs(att[t].reshape(HQ, D) - o) <= e).all(), t
        z = b["z"].to_numpy(np.float32, (T, K))
        quant, a = oracle.quantise_rows(att.astype(np.float32))
        assert (z == oracle.rescale(oracle.dense_i8(quant, self.w_o), a, 0.05)).all()
        want, e = op.adapters(att, slot, z.astype(np.float64), *self.lora[1])
        assert (np.abs(b["z1"].to_numpy(np.float32, (T, K)) - want) <= e).all()


def test_prompt_then_tokens():
    sp.device_init(0)
    st = sp.Stream()
    blk = Block(1)
    r = np.random.default_rng(2)
    lens = [37, 1, 130, 64]
    B = len(lens)
    blk.rows = B * CAP
    zero = np.zeros((blk.rows, HKV, D), np.uint16)
    blk.k, blk.v = sp.DeviceBuffer.from_numpy(zero), sp.DeviceBuffer.from_numpy(zero)
    start = np.arange(B, dtype=np.int32) * CAP

    def inputs(b, nq, done):
        T = int(np.sum(nq))
        xb, x64 = op.narrow(r.standard_normal((T, K)), T16)
        seq = np.repeat(np.arange(B), nq)
        slot = np.array([1, -1, 0, 2], np.int32)[seq]
        pos = np.concatenate([np.arange(d, d + n) for d, n in zip(done, nq)]).astype(np.int32)
        row = (start[seq] + pos).astype(np.int32)
        first = np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)
        length = (np.asarray(done) + nq).astype(np.int32)
        for n, v in (("x", xb), ("slot", slot), ("pos", pos), ("row", row), ("first", first), ("start", start), ("len", length)):
            b[n].upload(v)
        before = [op.widen(c.to_numpy(np.uint16, (blk.rows, HKV, D)), T16) for c in (blk.k, blk.v)]
        return T, x64, slot, pos, row, first, start, length, before

    print("prompt", flush=True)
    b = blk.buffers(sum(lens), B, max(lens), max(lens))
    args = inputs(b, np.array(lens), [0] * B)
    blk.issue(b, args[0], st)
    st.sync()
    blk.check(b, *args)

    print("tokens, as a graph", flush=True)
    c = blk.buffers(B, B, 1, CAP)
    done = list(lens)
    args = inputs(c, np.ones(B, int), done)
    with sp.Graph(st) as g:
        blk.issue(c, B, st)
    for step in range(4):
        print("replay", step, flush=True)
        args = inputs(c, np.ones(B, int), done)
        g.launch(st)
        st.sync()
        blk.check(c, *args)
        z = c["z1"].to_numpy(np.uint32, (B, K))
        blk.issue(c, B, st)  # the program's own eager work between the replays; the same inputs give the same bits
        st.sync()
        assert (c["z1"].to_numpy(np.uint32, (B, K)) == z).all()
        done = [d + 1 for d in done]
    g.destroy()
    st.destroy()
