"""The KV cache of a decoder that is built from a GGUF file through GgufFile: fp32, fp16 or 4-bit."""
from __future__ import annotations

import numpy as np
import pytest

import chatnet_b200 as cn
from chatnet_b200 import _native as N
from chatnet_b200 import configs as cf
from chatnet_b200.gguf import GgufFile
from chatnet_b200.llama import CudaLlamaModel, tensor_names
from tests import gguf_writer as gw
from tests.test_gpu_llama import small_dc

KINDS = [({}, N.KV_F32), ({"kv_f16": True}, N.KV_F16), ({"kv_q4": True}, N.KV_Q4),
         ({"kv_f16": True, "kv_q4": True}, N.KV_Q4)]


def write(path, dc):
    m = dc.model
    host = cf.host_tensors(dc)
    names = tensor_names(m.n_layers)
    types = [cf.tensor_type(dc, n) for n in names]
    gw.write_gguf(path, gw.llama_metadata(m), gw.llama_tensors(host, names, types, m))
    return host


@pytest.mark.parametrize("kw,kind", KINDS)
def test_config(tmp_path, kw, kind):
    write(tmp_path / "m.gguf", small_dc())
    with GgufFile(tmp_path / "m.gguf") as g:
        c = g.llama_config(max_batch=3, **kw)
    assert c.to_c().kv_dtype == kind and c.max_batch == 3


@pytest.mark.gpu
@pytest.mark.parametrize("kw,kind", KINDS)
def test_model(ctx, tmp_path, kw, kind):
    """The file's model and one built from its tensors give the same bits and hold the same rows."""
    dc = small_dc()
    dc = cf.replace(dc, model=cf.replace(dc.model, **kw), kv_filled=0, decode_pos=0)
    host = write(tmp_path / "m.gguf", dc)
    with GgufFile(tmp_path / "m.gguf") as g:
        a = g.llama_model(ctx, max_batch=1, **kw)
    ts = cf.device_tensors(ctx, dc, host)
    b = CudaLlamaModel(ctx, dc.model, ts)
    toks = [5, 77, 401, 12]
    for pos, t in enumerate(toks):
        np.testing.assert_array_equal(a.forward([t], pos), b.forward([t], pos))
    for layer in range(dc.model.n_layers):
        for x, y in zip(a.kv_read(0, layer, 0, 4), b.kv_read(0, layer, 0, 4)):
            assert x.dtype == (np.float16 if kind == N.KV_F16 else np.float32) and x.any()
            np.testing.assert_array_equal(x, y)
    x = a.kv_read(0, 0, 0, 4)[0].astype(np.float64).reshape(-1, 32)
    steps = np.unique(np.round(x / np.abs(x).max(-1, keepdims=True) * 8 * 4)).size  # (levels: multiples of an eighth)
    assert (steps <= 24) if kind == N.KV_Q4 else (steps > 24)
    a.close()
    b.close()
    for t in ts:
        t.free()
