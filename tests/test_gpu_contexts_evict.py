"""GPU tests of eviction (include/bitserve.h) at the ends of its numbers' ranges, against
context_ref.evict bit for bit."""
import numpy as np
import pytest
import torch

import serve_ref as ref
from test_gpu_contexts import check_evict, random_account

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

MOST = 2 ** 31 - 1


@pytest.mark.filterwarnings("ignore:overflow")  # 2^31 on the way to shift + size - keep
@pytest.mark.parametrize("size,keep", [(20, 10), (9000, 4000)])
@pytest.mark.parametrize("recent", [0, 1, 3, MOST])
@pytest.mark.parametrize("sink", [0, -5, MOST])
@pytest.mark.parametrize("end", ["first", "last"])
def test_tokens_at_the_ends_of_int32(size, keep, recent, sink, end):
    """The last token is 2^31 - 1, or the first -2^31: recent ones are those from len + shift - recent on, also
    where that is 2^31 or below -2^31."""
    rng = np.random.default_rng(size)
    table, n_pages = ref.pages_for([(0, size)] * 2, 16, rng)
    cache = ref.rand_cache(rng, n_pages, 2, 16, 16)
    account = list(random_account(rng, [size] * 2, 2, size + 1, [0, 0], False))
    account[0][:, :, size - 1] = -1e30  # the last position goes where nothing keeps it
    account[3][:] = MOST - (size - 1) if end == "last" else -2 ** 31
    check_evict(cache, table, [size] * 2, account, [keep] * 2, [sink] * 2, [recent] * 2)
