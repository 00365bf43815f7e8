"""Limits of the paged 4-bit cache that are refused on the host, and the calls that carry a resize's grants."""

import pytest

from tests.test_kv_cache_cpu import ATTEND, RESIZE, STEP, A, lib  # noqa: F401 -- lib is a fixture
from torchnative_b200 import _native as N


@pytest.mark.parametrize("page", [16, 64, 1024])
def test_a_row_of_the_table_names_at_most_2_to_the_31_less_1024_tokens(lib, page):  # noqa: F811
    """32-bit positions: a tile of keys behind the last one has to stay below 2^31."""
    most = (2**31 - 1024) // page
    for args, op in ((RESIZE, "tn_kv_pages_resize"), (ATTEND, "tn_sdpa_q4_cache"), (STEP, "tn_sdpa_q4_decode_step")):
        for pages, want in ((most + 1, N.TN_ERR_SHAPE), (most, N.TN_ERR_INVALID)):  # the latter: for its null table
            call = {**args, "page": page, "max_pages": pages, "stride": pages, "table": None}
            assert getattr(lib, op)(*call.values(), None) == want, (op, pages)
            assert op in N.last_error()


def test_grants_change_no_refusal(lib):  # noqa: F811
    for change, status in ((dict(page=24), N.TN_ERR_NOT_IMPLEMENTED), (dict(requests=-1), N.TN_ERR_SHAPE),
                           (dict(lengths=None), N.TN_ERR_INVALID), (dict(new=A), N.TN_ERR_INVALID)):
        assert lib.tn_kv_pages_resize_granted(*{**RESIZE, **change}.values(), A, None) == status
    for change, status in ((dict(heads=72), N.TN_ERR_NOT_IMPLEMENTED), (dict(rows=0), N.TN_ERR_SHAPE),
                           (dict(qkv=None), N.TN_ERR_INVALID), (dict(ws_bytes=0), N.TN_ERR_SHAPE)):
        assert lib.tn_sdpa_q4_decode_step_granted(*{**STEP, **change}.values(), A, None) == status
    assert lib.tn_sdpa_q4_decode_step_granted(*{**STEP, "requests": 0}.values(), A, None) == N.TN_OK
    assert lib.tn_llama_argmax_embed_granted(A, 0, 100, A, A, 64, A, None, A, None) == N.TN_OK
