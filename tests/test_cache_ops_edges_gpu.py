"""Keys and values in 8 bits and attention of shared prefixes at the edges of what their entries take: starts that are only as aligned as the header
asks, more rows than one launch holds, one key that leads far in front of a long flat history.  Bounds as in tests/test_cache_ops_gpu.py."""
import numpy as np
import pytest
import torch

from tests import _gpu_util as G
from tests._gpu_util import DEV, check, dev_i32, lib, ptr, sync
from tests.test_cache_ops_gpu import Cache

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ read-back
@pytest.mark.parametrize("d,page,off", [(64, 16, 8), (128, 64, 8), (128, 8, 24), (64, 32, 16)])
def test_read_into_a_pool_that_starts_on_16_bytes(d, page, off):
    """The bf16 pool starts `off` entries behind a 256-byte boundary: on 16 bytes as the header asks, and only off = 16 on 32."""
    ctx, nkv = [1, 100, page, 0, 3 * page + 5], 3
    c = Cache(ctx, nkv, d, page, 7)
    area = G.empty((c.n_pages * 2 * nkv * page * d + 32,), torch.bfloat16)
    area.zero_()
    back = area[off:off + c.n_pages * 2 * nkv * page * d].view(c.n_pages, 2, nkv, page, d)
    assert back.data_ptr() % 16 == 0 and (back.data_ptr() % 32 == 0) == (off % 16 == 0)
    check(lib().dis_k_kv_read_i8(ptr(c.pool), ptr(c.scale), ptr(back), ptr(c.d_table), ptr(c.d_table), c.width, ptr(dev_i32(np.arange(len(ctx)))), None,
                                 ptr(dev_i32(ctx)), len(ctx), nkv, d, page, None))
    sync()
    used = c.used.to(DEV)[:, None, None, :, None].expand(back.shape)
    want = torch.where(used, c.value.float().to(torch.bfloat16), torch.zeros((), dtype=torch.bfloat16, device=DEV))
    assert torch.equal(back, want)
    assert int((area[:off] != 0).sum()) == 0 and int((area[off + back.numel():] != 0).sum()) == 0
