"""Tensor-parallel ranks on a 4-bit KV cache: each holds its kv heads' rows; the ranks' logits are the same bits and
match LlamaModel.Forward over the rows that all of them hold.  More than one rank needs as many GPUs."""
from __future__ import annotations

import multiprocessing as mp

import numpy as np
import pytest
import torch

import chatnet_b200 as cn
from chatnet_b200 import configs as cf
from tests.parity import REL_TOL, rel_err
from tests.test_gpu_kvq4_model import NumpyLlama, q4_dc

pytestmark = pytest.mark.gpu

STEPS = 3


def tp_dc():
    dc = q4_dc(head_dim=64, n_heads=8, n_kv=2, ctx_len=40)
    return cf.replace(dc, model=cf.replace(dc.model, hidden_dim=1024, vocab=512), kv_filled=20, decode_pos=20)


def rank_main(rank, size, dc, to_parent, from_parent):
    import ctypes as C

    from chatnet_b200 import _native as N
    from chatnet_b200.llama import CudaLlamaModel
    try:
        ctx = cn.Context(rank)
        m = dc.model
        tp = cn.TensorParallel(ctx, rank, size, m.max_batch, m.dim, m.vocab)
        to_parent.put(("handle", rank, tp.ipc_handle()))
        tp.connect(from_parent.get(timeout=120))
        ts = cf.device_tensors(ctx, dc, cf.host_tensors(dc), rank=rank, size=size)
        model = CudaLlamaModel(ctx, m, ts, tp=tp)
        model.kv_synth(0, dc.kv_filled, *cf.kv_seeds(dc, 0))
        model.prepare(1)
        to_parent.put(("ready", rank, None))
        assert from_parent.get(timeout=120) == "go"
        outs = [model.decode([cf.token(dc, 0, s)], [dc.decode_pos + s])[0].copy() for s in range(STEPS)]
        n, own = dc.decode_pos + STEPS, m.kv_dim // size  # this rank's columns of the rows
        rows = np.empty((m.n_layers, 2, n, own), np.float32)
        for l in range(m.n_layers):
            k, v = (rows[l, i].ctypes.data_as(C.c_void_p) for i in range(2))
            cn.check(N.lib().cn_llama_kv_read(model.handle, 0, l, 0, n, k, v), "cn_llama_kv_read")
        model.close()
        for t in ts:
            t.free()
        tp.close()
        ctx.close()
        to_parent.put(("done", rank, (outs, rows)))
    except Exception as e:  # reported to the parent, which fails the test
        to_parent.put(("error", rank, repr(e)))


def run_group(dc, size):
    ctx = mp.get_context("spawn")
    to_parent, to_child = ctx.Queue(), [ctx.Queue() for _ in range(size)]
    procs = [ctx.Process(target=rank_main, args=(r, size, dc, to_parent, to_child[r]), daemon=True)
             for r in range(size)]
    for p in procs:
        p.start()
    try:
        def collect(kind):
            got = {}
            while len(got) < size:
                k, r, v = to_parent.get(timeout=300)
                assert k == kind, (k, r, v)
                got[r] = v
            return [got[r] for r in range(size)]
        handles = collect("handle")
        for q in to_child:
            q.put(handles)
        collect("ready")
        for q in to_child:
            q.put("go")
        return collect("done")
    finally:
        for p in procs:
            p.join(timeout=60)
            if p.is_alive():
                p.kill()


@pytest.mark.parametrize("size", [1, 2])
def test_ranks_decode(oracle, size):
    if torch.cuda.device_count() < size:
        pytest.skip(f"needs {size} GPUs")
    dc = tp_dc()
    res = run_group(dc, size)
    for outs, _ in res[1:]:
        for a, b in zip(outs, res[0][0]):
            np.testing.assert_array_equal(a, b)
    rows = np.concatenate([r[1] for r in res], -1)

    class Held:
        def kv_read(self, seq, layer, pos0, npos):
            return rows[layer, 0, pos0:pos0 + npos], rows[layer, 1, pos0:pos0 + npos]
    ref = NumpyLlama(oracle, dc, cf.host_tensors(dc))
    for s in range(STEPS):
        want = ref.forward(Held(), [cf.token(dc, 0, s)], dc.decode_pos + s)[-1]
        assert rel_err(res[0][0][s][0], want) <= REL_TOL, s
