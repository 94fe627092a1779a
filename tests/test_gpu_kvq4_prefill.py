"""Scores of texts that run as one prefill pass, on a 4-bit and an fp32 KV cache, and the launches of such a pass."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from chatnet_b200 import _native as N
from chatnet_b200 import configs as cf
from tests.parity import REL_TOL
from tests.test_gpu_kvq4_model import build, q4_dc  # noqa: F401
from tests.test_gpu_llama import small_dc

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def check_scores(lp, ent, logits, nxt):
    """Against the logits in 64 bits, each of which may be off by t = 1e-3 of the largest: a log probability by 2 t, an
    entropy, whose gradient is p |log p + H| in sum at most 2 H, by 2 t (H + 1)."""
    want = torch.log_softmax(torch.from_numpy(logits), -1).numpy()
    h = -(np.exp(want) * want).sum(-1)
    t = REL_TOL * np.abs(logits).max(-1)
    assert (np.abs(lp - want[np.arange(len(nxt)), nxt]) <= 2 * t).all()
    assert (np.abs(ent - h) <= 2 * t * (h + 1)).all()


@pytest.mark.parametrize("head_dim,n_heads,n_kv,neox", [(64, 4, 2, False), (128, 2, 1, True)])
def test_score_4_bit_cache(build, head_dim, n_heads, n_kv, neox):  # noqa: F811
    """A text whose head runs in several batches of rows, a second piece behind it, and a short one by decode steps;
    each attends over what the cache holds."""
    dc = q4_dc(head_dim, n_heads, n_kv, neox=neox, ctx_len=200)
    g, r = build(dc)
    toks = np.random.default_rng(2).integers(0, dc.model.vocab, 140)
    g.set_prefill(16)
    for lo, hi in ((0, 70), (69, 120), (119, 130)):  # (a text's last token is scored, not run)
        lp, ent = g.score(toks[lo:hi], lo)
        check_scores(lp, ent, r.forward(g, toks[lo:hi - 1], lo), toks[lo + 1:hi])


def test_score_fp32_cache(build):  # noqa: F811
    dc = cf.replace(small_dc(ctx_len=100), kv_filled=0, decode_pos=0)
    g, _ = build(dc)
    toks = np.random.default_rng(1).integers(0, dc.model.vocab, 80)
    g.set_prefill(0)
    logits = np.stack([g.forward([int(t)], i) for i, t in enumerate(toks[:-1])]).astype(np.float64)
    g.set_prefill(16)
    for lo, hi in ((0, 50), (49, 80)):
        lp, ent = g.score(toks[lo:hi], lo)
        check_scores(lp, ent, logits[lo:hi - 1], toks[lo + 1:hi])


def test_entropies_are_optional(build):  # noqa: F811
    g, _ = build(q4_dc(ctx_len=100))
    toks = np.random.default_rng(3).integers(0, 500, 60).astype(np.int32)
    for least in (0, 16):
        g.set_prefill(least)
        want, _ = g.score(toks)
        lp = np.full(60, 7.5, np.float32)
        assert N.lib().cn_llama_score(g.handle, toks.ctypes.data, 60, 0, lp.ctypes.data, None) == 0
        np.testing.assert_array_equal(lp[:59], want)
        assert lp[59] == 7.5


def kernel_nodes(graph):
    cu = C.CDLL("libcuda.so.1")
    h, n = C.c_void_p(graph.raw_cuda_graph()), C.c_size_t(0)
    assert cu.cuGraphGetNodes(h, None, C.byref(n)) == 0
    nodes = (C.c_void_p * n.value)()
    assert cu.cuGraphGetNodes(h, nodes, C.byref(n)) == 0
    kinds = []
    for v in nodes:
        k = C.c_int(-1)
        assert cu.cuGraphNodeGetType(C.c_void_p(v), C.byref(k)) == 0
        kinds.append(k.value)
    return kinds.count(0)  # CU_GRAPH_NODE_TYPE_KERNEL


def test_kernels_of_a_prefill_pass(ctx, build):  # noqa: F811
    dc = q4_dc(ctx_len=100)
    g, _ = build(dc)
    x = torch.randn(40, dc.model.dim, device="cuda")
    out = torch.empty_like(x)
    torch.cuda.synchronize()
    g.prefill_hidden_dev(x.data_ptr(), 40, 0, out.data_ptr())  # (the first pass makes its buffers)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(ctx.stream)):
        g.prefill_hidden_dev(x.data_ptr(), 40, 0, out.data_ptr())
    assert kernel_nodes(graph) == g.prefill_kernels()
    graph.reset()
