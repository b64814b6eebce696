"""``PagedKVCache``'s sizes, on the CPU."""

from __future__ import annotations

import pytest

from flux_b200.paged import PagedKVCache

SMALL = dict(layers=1, pages=1, kv_heads=1, head_dim=8, sequences=1, max_rows=1, page_size=1, device="meta")


@pytest.mark.parametrize("change", [{"pages": 2 ** 20 + 1}, {"sequences": 2 ** 18 + 1}, {"kv_heads": 65536},
                                    {"page_size": 65537}, {"max_rows": 2 ** 31}, {"max_rows": 2 ** 31 - 1, "page_size": 16}])
def test_sizes_that_no_operator_takes_are_refused(change):
    with pytest.raises(ValueError, match="at most"):
        PagedKVCache(**{**SMALL, **change})


@pytest.mark.parametrize("change,columns", [({"pages": 2 ** 20}, 1), ({"sequences": 2 ** 18}, 1), ({"kv_heads": 65535}, 1),
                                            ({"page_size": 65536}, 1), ({"max_rows": 2 ** 31 - 1}, 2 ** 31 - 1),
                                            ({"max_rows": 100, "page_size": 16}, 7)])
def test_sizes_up_to_the_limits(change, columns):
    assert PagedKVCache(**{**SMALL, **change}).page_table.shape[1] == columns
