"""Which kernel paged attention runs on (csrc/dispatch.hpp), asked on the CPU: most
shapes below were timed with the kernels on an MI355X, and the rule takes the
fastest one for most contexts (the lengths are on the device)."""
import os

import pytest

from gpu_util import dispatch_rules, nnhip
from test_paged import OPS


@pytest.fixture(scope="module")
def rules():
    return dispatch_rules()


@pytest.mark.parametrize("T,B,G,Hkv,want", [
    # prompts that fill the card with units of 128 columns
    (3400, 4, 4, 4, "tall"), (8000, 1, 4, 8, "tall"), (1700, 4, 4, 4, "tall"),
    (768, 4, 8, 4, "tall"), (2050, 16, 4, 4, "tall"), (10 ** 8, 1, 32, 8, "tall"),
    # fewer rows, requests that do not fill a unit, decoding ones among prompts
    (512, 1, 4, 4, "short"), (900, 4, 4, 4, "short"), (1030, 33, 4, 4, "short"),
    (2200, 100, 4, 4, "short"), (1, 1, 1, 1, "short"), (32, 32, 4, 8, "short"),
    (128, 128, 4, 8, "short"), (0, 5, 1, 1, "short"), (50, 4096, 1, 1, "short"),
    # many units of single tokens
    (439, 512, 1, 16, "solo"), (439, 512, 4, 4, "solo"), (1600, 1600, 1, 1, "solo"),
    (4096, 4096, 8, 8, "solo"), (100, 100, 3, 16, "solo")])
def test_paged_attention(rules, T, B, G, Hkv, want):
    got = "tall" if rules.attention_paged_tall(T, B, G, Hkv) else \
        "solo" if rules.attention_paged_solo(T, B, G, Hkv) else "short"
    assert got == want


@pytest.mark.skipif(not os.path.exists(nnhip.LIB_PATH), reason="libnnhip.so not built")
@pytest.mark.parametrize("op", ["nnhip_rope_kv_append_paged_q8", "nnhip_attention_paged_q8",
                                "nnhip_kv_read_paged_q8"])
def test_a_pool_of_more_heads_than_are_counted_is_refused(op):
    good = dict(OPS[op], num_blocks=2 ** 20, Hkv=1024)
    if "H" in good:
        good["H"] = 1024
    with pytest.raises(nnhip.NNHipError, match="num_blocks") as e:
        nnhip.call(op, *good.values())
    assert e.value.code == nnhip.EARG
    good["num_blocks"] = 2 ** 20 - 1              # as many as there may be: the next check
    with pytest.raises(nnhip.NNHipError, match="NULL"):
        nnhip.call(op, *good.values())
