"""A prompt's MLP over 8-bit weights whose down product the defaults split along
K: a longer block beside a recorded graph of a shorter one."""
import numpy as np
import pytest

import f8_ref as f8
import herbert_hip as hb
from st_writer import write_model

pytestmark = pytest.mark.gpu


def test_graph_of_a_short_block(tmp_path):
    """On a context of its own, whose workspace nothing else has grown."""
    h, inter, short, n = 512, 4608, 40, 500
    gate, up = hb.normal_bf16(81, 0.02, (inter, h)), hb.normal_bf16(82, 0.02, (inter, h))
    down, pn = hb.normal_bf16(83, 0.02, (h, inter)), hb.normal_bf16(84, 0.1, (h,))
    p = "model.language_model.layers.0."
    write_model(str(tmp_path / "m"), [{p + "mlp.gate_proj.weight": ("BF16", gate), p + "post_attention_layernorm.weight": ("BF16", pn),
                                       p + "mlp.up_proj.weight": ("BF16", up), p + "mlp.down_proj.weight": ("BF16", down)}])
    x0 = hb.normal_bf16(85, 1.0, (n, h))
    gpu = hb.Gpu(0)
    try:
        with hb.Checkpoint(str(tmp_path / "m")) as ck, hb.Engine(gpu, "prefill.block=512") as e:
            mlp = hb.PrefillMlp(gpu, e, ck, 0, h, inter, f8=True)
        names = {m: gpu.kernel_name(k[2]) for m, k in mlp.kern.items()}
        assert all("_ks" in s for s in names.values()), names
        X, Y = gpu.alloc_with(x0[:short]), gpu.alloc_with(x0)
        few, many = mlp.states(short), mlp.states(n)
        gpu.time_ops(mlp.ops(X, short, few), 1)
        want = gpu.download(X, np.uint16, short * h)
        graph = gpu.graph(mlp.ops(X, short, few))
        for _ in range(3):
            gpu.upload(X, x0[:short])
            graph.launch()
            gpu.sync()
            assert np.array_equal(gpu.download(X, np.uint16, short * h), want)
            # The longer block, whose slabs are larger.
            gpu.upload(Y, x0)
            gpu.time_ops(mlp.ops(Y, n, many), 1)
            got = gpu.download(Y, np.uint16, n * h).reshape(n, h)
            raw = gpu.download(mlp.buf["h8"], np.uint8, n * hb.f8_row_bytes(inter))
            hv, wv = f8.row_values(*f8.unpack_rows(raw, n, inter)), f8.values(*f8.quantize(down))
            y = hv @ wv.T + f8.f64(x0)
            f8.close(got, y, f8.mfma_bound(hv, wv) + f8.U * np.abs(y), "down")
        graph.free()
    finally:
        gpu.close()
