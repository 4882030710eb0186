"""The experts' 8-bit kernels over tables whose count of tiles is more than the
table holds, or than a launch's pairs: no entry past its end is looked at."""
import numpy as np
import pytest

import f8_ref as f8
import herbert_hip as hb
from test_gpu_f8 import Bufs, marked, run
from test_gpu_f8_gemm import tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bm", [16, 32, 64])
@pytest.mark.parametrize("t", [1, 3, 40])
def test_counts_past_the_table(gpu, bm, t):
    inter, hidden, top_k, experts = 128, 272, 2, 6
    rng = np.random.default_rng(bm + t)
    flat, order, tiles = tables(rng, t, top_k, experts, bm, False)
    w = [f8.exact_weights(rng, hidden, inter) for _ in range(experts)]
    pairs = t * top_k
    x = f8.exact_x(rng, pairs, inter)
    got = {}
    with Bufs(gpu) as b:
        st, ls, wr = b.put(np.array([0, 0, 0, t], np.uint32)), b.put(order), b.put(np.concatenate([f8.pack(*v) for v in w]))
        xr = b.put(x if bm == 16 else f8.pack_rows(*f8.quantize_rows(x)))
        for count in (tiles[0], len(tiles) // 3, len(tiles) // 3 + 1, 1 << 20, 0x55555556, 0xFFFFFFFF):
            tab = tiles.copy()
            tab[0] = count
            # Behind the table, what would be a tile of the first expert.
            tl, y = b.put(np.concatenate([tab, np.array([0, 0, 1] * 8, np.uint32)])), b.put(marked((pairs, hidden), np.uint16))
            tl.size = tab.nbytes
            run(gpu, hb.experts_f8(inter, hidden, hb.Out.Bf16, hb.Rows.Scatter, top_k, experts, t, bm), [st, wr, xr, y, ls, tl], t)
            got[int(count)] = b.get(y, np.uint16, (pairs, hidden))
    want = np.zeros((pairs, hidden))
    for p in range(pairs):
        want[order[p]] = f8.f64(x[p]) @ f8.values(*w[flat[order[p]]]).T
    for count, y in got.items():
        assert np.array_equal(y, hb.f32_to_bf16(want.astype(np.float32))), count
