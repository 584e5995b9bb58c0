"""Refusals of the step of rows that share blocks, on the host before any launch (no GPU here)."""

import pytest

from tests.test_loop_abi import INV, P, call, refused

ST = dict(bt=P, bts=8, rb=P, pos=P, sh=P, nb=100, fin=None, ring=P, state=P, cap=100, bs=16, slots=P,
          lens=P, status=P, rows=6, stream=None)


@pytest.mark.parametrize("over,needle", [
    (dict(sh=None), "shared"), (dict(nb=0), "num_blocks"), (dict(nb=-1), "num_blocks"),
    (dict(rows=-1), "num_rows"), (dict(bts=-1), "block_table_stride"), (dict(cap=0), "free_ring_capacity"),
    (dict(bt=None), "non-null"), (dict(rb=None), "non-null"), (dict(ring=None), "non-null"),
    (dict(state=None), "non-null"), (dict(bs=0), "block_size"), (dict(status=None), "status"),
    (dict(pos=None), "positions"), (dict(slots=None), "slot_mapping"), (dict(lens=None), "context_lens"),
])
def test_step_rejects(over, needle):
    refused("vpa_decode_step_metadata_shared", ST, over, INV, needle)
    if not {"sh", "nb"} & set(over):
        old = {k: v for k, v in ST.items() if k not in ("sh", "nb")}
        code, message = call("vpa_decode_step_metadata", old, over)
        assert code == INV and "decode_step_metadata:" in message
