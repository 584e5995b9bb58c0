"""The workspace of paged_attention_weights by the sizes of a call (CPU): logits are stored
only where a (sequence, kv head) has at most 16 rows."""

import pytest

import vpa
from vpa import _lib
from tests.test_loop_abi import INV, P, WS, WT, refused


def at_most(rows, h, ctx):
    return _lib.load().vpa_paged_attention_weights_workspace_size(rows, h, ctx)


def of_call(rows, mq, ctx, h, kvh):
    return _lib.load().vpa_paged_attention_weights_call_workspace_size(rows, mq, ctx, h, kvh)


@pytest.mark.parametrize("rows,mq,ctx,h,kvh", [(256, 32, 6000, 16, 8), (8192, 8192, 8192, 16, 8),
                                               (30000, 30000, 30000, 16, 8), (17, 17, 300, 1, 1),
                                               (1, 1, 5, 17, 1), (9, 3, 257, 12, 2)])
def test_rows_of_a_prompt_keep_a_pair_per_chunk(rows, mq, ctx, h, kvh):
    assert mq * (h // kvh) > 16
    assert of_call(rows, mq, ctx, h, kvh) == rows * h * -(-ctx // 256) * 8
    # over 4096 tokens half of what the rows themselves hold, at 128 dims of 16 bits
    assert of_call(rows, mq, 4096, h, kvh) == rows * h * 256 // 2


@pytest.mark.parametrize("rows,mq,ctx,h,kvh", [(256, 1, 4096, 16, 8), (24, 8, 6000, 16, 8),
                                               (3, 1, 1, 16, 1), (40, 16, 257, 4, 4)])
def test_few_rows_keep_their_logits(rows, mq, ctx, h, kvh):
    assert of_call(rows, mq, ctx, h, kvh) == at_most(rows, h, ctx) == rows * h * -(-ctx // 256) * 1032


def test_nothing():
    for args in ((0, 3, 5, 16, 8), (4, 0, 5, 16, 8), (4, 3, 0, 16, 8), (4, 3, 5, 0, 8), (4, 3, 5, 16, 0)):
        assert of_call(*args) == 0
    assert of_call(1 << 20, 1 << 18, 1 << 28, 64, 8) == (1 << 20) * 64 * (1 << 20) * 8  # in 64 bits


@pytest.mark.parametrize("over", [dict(mq=9), dict(mq=3), dict(mq=1, cu=None, rows=4)])
def test_a_byte_less_is_refused(over):
    a = {**WT, **over}
    need = of_call(a["rows"], a["mq"], a["mc"], a["h"], a["kvh"])
    refused("vpa_paged_attention_weights", WT, {**over, "wsb": need - 1}, WS, f"{need} bytes needed")
    refused("vpa_paged_attention_weights", WT, {**over, "ws": None}, WS, f"{need} bytes needed")
    refused("vpa_paged_attention_weights", WT, {**over, "wsb": need, "ws": P + 128}, INV, "256-byte")


def test_python_helper():
    def size(*a, **kw):
        t = vpa.paged_attention_weights_workspace(*a, "cpu", **kw)
        return None if t is None else t.numel()

    assert size(256, 16, 6000) == at_most(256, 16, 6000)
    assert size(256, 16, 6000, max_query_len=32, num_kv_heads=8) == of_call(256, 32, 6000, 16, 8)
    assert size(256, 16, 6000, max_query_len=8, num_kv_heads=8) == at_most(256, 16, 6000)
    assert size(0, 16, 6000) is None and size(0, 16, 6000, max_query_len=32, num_kv_heads=8) is None
