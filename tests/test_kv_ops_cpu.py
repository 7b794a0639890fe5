"""CPU-side checks of the operators over the KV cache: their entry points
refuse null and stale contexts with a message, before anything is read, and
the ctypes mirrors have the header's layout."""
import ctypes as C

import pytest

from vxg_amd import engine

CALLS = {
    "vxt_hip_attn_tree_q8_dev": [None, None, 4, None, 1, 0, None, None, None],
    "vxt_hip_attn_tree_step_q8_dev": [None, None, None, 0, None, None, 0, None, 1, 0, 0, None, None],
    "vxt_hip_kv_q8_keep_path_dev": [None, None, 1, 0, None],
    "vxt_hip_attn_weigh_q8_dev": [None, None, None, 4, 1, 0, 0, None, None, None],
    "vxt_hip_kv_q8_evict_dev": [None, None, 1, 1, 1, 0, 0, None, None, None],
    "vxt_hip_kv_q8_block_means_dev": [None, None, 0, 1, None],
    "vxt_hip_attn_blocks_q8_dev": [None, None, None, 4, 1, 0, 1, 0, 1, None, None, None, None],
}


@pytest.mark.parametrize("name", sorted(CALLS))
@pytest.mark.parametrize("ctx", [None, 0x1000])
def test_contexts_that_are_not_live_are_refused(name, ctx):
    lib = engine.load_library()
    buf = C.create_string_buffer(256)
    rc = getattr(lib, name)(ctx, *CALLS[name], buf, len(buf))
    assert rc == engine.VXT_E_ARG and buf.value


def test_struct_layouts():
    assert C.sizeof(engine.KvWeightsView) == 24 and engine.KvWeightsView.max_seq.offset == 16
    assert C.sizeof(engine.KvBlockMeansView) == 24 and engine.KvBlockMeansView.block.offset == 20
