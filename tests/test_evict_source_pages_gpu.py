"""Eviction from pages that rows certainly come from and that are no pages of the cache."""
import pytest
import torch

from jit_kernel import _native
from jit_kernel.topk_indexer import _status_word, kernel_status
from test_cache_evict_gpu import check, make, take_status, weights
from test_paged_attention_gpu import gen

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def status():
    if torch.cuda.is_available():
        _status_word(torch.device("cuda", 0)).zero_()
    yield
    if torch.cuda.is_available():
        assert kernel_status() == 0


@pytest.mark.parametrize("dtype,D", [(FP8, 128), (torch.bfloat16, 128), (torch.float16, 24)])
@pytest.mark.parametrize("recent,sinks", [(60, 4), (8, 4)])
@pytest.mark.parametrize("page", [0, 9])  # (of 10: the first rows, and the last ones)
@pytest.mark.parametrize("entry", ["-1", "-2147483648", "behind", "far"])
def test_source_pages_that_do_not_exist(entry, page, recent, sinks, dtype, D):
    """The places their rows would go to stay as they are, whatever else moves."""
    g = gen(page + recent)
    data, scales, table, to = make(g, [160], 64, 2, D, 16, dtype)
    table[0, page] = {"behind": data[0].size(0) // 16, "far": 0x7fffffff}[entry] if entry in ("behind", "far") else int(entry)
    check(data, scales, table, to, weights(g, 1, 2, 160), [160], 16, 64, recent, sinks)
    assert take_status() == _native.ST_BAD_INDEX


@pytest.mark.parametrize("dtype", [FP8, torch.bfloat16])
@pytest.mark.parametrize("entry", ["-1", "behind", "far"])
def test_a_source_page_between_the_protected_rows(entry, dtype):
    """Rows that stay for their weight: nearly all of page 3's."""
    g = gen(3)
    data, scales, table, to = make(g, [160], 64, 2, 128, 16, dtype)
    w = weights(g, 1, 2, 160)
    w[..., 48:60] += 1e6
    table[0, 3] = {"-1": -1, "behind": data[0].size(0) // 16, "far": 0x7fffffff}[entry]
    kept, _, _ = check(data, scales, table, to, w, [160], 16, 64, 8, 4)
    assert bool(((kept >= 48) & (kept < 60)).sum(2).eq(12).all())
    assert take_status() == _native.ST_BAD_INDEX
