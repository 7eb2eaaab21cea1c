"""The borders that the tests of few kv heads look at are the library's."""
import os
import re

from test_gpu_pages_heads import CASES
from test_launch_order_cpu import CSRC


def test_borders():
    text = open(os.path.join(CSRC, "pages_shared.cuh")).read()
    assert {n: int(v) for n, v in re.findall(r"PST_(MIN_ROWS|MIN_PAGES|ALL_ROWS|ALL_WORK) = (\d+)", text)} == {"MIN_ROWS": 640, "MIN_PAGES": 32, "ALL_ROWS": 1024, "ALL_WORK": 95000}
    for heads_kv, group, n_tok, pages, images in CASES:
        assert images == (n_tok * group > 640 and n_tok * group * heads_kv > 1024 and pages >= 32 and n_tok * group * heads_kv * pages * heads_kv >= 95000)
    assert sum(x[-1] for x in CASES) > 8
