"""kv_append and kv_read with a bound of rows far above the rows of the call."""
import numpy as np
import pytest

import decode_ref as R
import viper_amd as va
from test_gpu_kv_cache import SENT, back, dev, gpu_cache, table_for

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("max_rows", [2 ** 31 - 1, 2 ** 31 - 31, 2 ** 24, 40])
@pytest.mark.parametrize("D", [64, 128])
def test_any_bound_of_rows(max_rows, D):
    rng = np.random.default_rng(40)
    kvh, page, lens, counts = 3, 32, [70, 33, 40], [40, 0, 7]
    print(f"max_rows={max_rows} D={D}", flush=True)
    table, pages = table_for(rng, lens, page)
    offs = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    g = gpu_cache(R.Cache(False, pages, page, kvh, D))
    batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), max_rows, dev(offs))
    k, v = (R.bf16_bits(rng.standard_normal((48, kvh * D))) for _ in range(2))  # a row behind the last sequence's
    ko, vo = (dev(np.full((48, kvh, D), SENT)) for _ in range(2))
    assert va.kv_append(g, batch, dev(k), dev(v)).ok() and va.kv_read(g, batch, ko, vo).ok()
    for got, want in ((back(ko), k), (back(vo), v)):
        np.testing.assert_array_equal(got.reshape(48, -1)[:47], want[:47])
        assert np.all(got[47] == SENT)
