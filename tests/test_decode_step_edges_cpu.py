"""Sizes of the decode step's operators next to 2^31 that their 32-bit indexes do not hold are refused, without a GPU."""
import pytest

from test_decode_step_cpu import _refused, _rope, capi  # noqa: F401


@pytest.mark.parametrize("batch,cols", [(1, 0x7fffffff), (1, 0x7fffffff - 65535), (16383, 131080), (2, 1 << 30)])
def test_tables_next_to_32_bits_are_refused(capi, batch, cols):  # noqa: F811
    f = dict(batch=batch, page_size=1, table_cols=cols, table_stride=cols, block_table=1 << 20, new_tokens=2 << 20, held=3 << 20, free_pages=4 << 20, free_capacity=9,
             free_count=5 << 20, total_tokens=2, cu_tokens=6 << 20, start=7 << 20, kv_len=8 << 20, positions=9 << 20, slots=10 << 20, free_count_out=11 << 20)
    _refused(capi, "lcml_kv_plan", capi.KvPlanDesc(**f))


@pytest.mark.parametrize("bad", [dict(q_heads=0x7fffffff), dict(k_heads=0x7fffffff - 30), dict(q_heads=0x7fffffff - 65535)])
def test_heads_next_to_32_bits_are_refused(capi, bad):  # noqa: F811
    f = dict(tokens=1, head_dim=2, rotary=2, q_token_stride=2, k_token_stride=2, q_head_stride=2, k_head_stride=2, q_out_head_stride=2, k_out_head_stride=2)
    _refused(capi, "lcml_qk_norm_rope", _rope(capi, **{**f, **bad}))
