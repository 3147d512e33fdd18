"""Packed weights in a state dict: what tells their scale layout apart is checked on the way in (no GPU)."""
import pytest
import torch

from rtx_b200.formats import (PACKED_OPERAND_SCHEMA_VERSION, SCALE_LAYOUT_CODES, mxfp8_state_for_kernel,
                              scales_row_major_to_mma128)


def state(layout, rows, k, *, version=PACKED_OPERAND_SCHEMA_VERSION, in_features=None):
    kp = (k + 31) // 32 * 32
    gen = torch.Generator().manual_seed(rows + k)
    row_major = torch.randint(100, 130, (rows, kp // 32), dtype=torch.uint8, generator=gen)
    tiles = scales_row_major_to_mma128(row_major, rows, kp // 32, (kp // 32 + 3) // 4)
    return {"a.weight_data": torch.zeros(rows, kp, dtype=torch.uint8),
            "a.weight_scales": row_major.reshape(-1) if layout == "row_major" else tiles,
            "a.weight_packing_meta": torch.tensor([version, SCALE_LAYOUT_CODES[layout], in_features or k, kp])}, tiles


@pytest.mark.parametrize("rows,k", [(128, 128), (256, 512), (200, 72), (384, 33)])
@pytest.mark.parametrize("layout", ["row_major", "mma128"])
def test_scales_become_tiles(rows, k, layout):
    held, tiles = state(layout, rows, k)
    first = held["a.weight_packing_meta"].clone()
    meta = held["a.weight_packing_meta"]
    assert mxfp8_state_for_kernel(held, "a.", rows, k) is None
    assert torch.equal(held["a.weight_scales"], tiles)
    assert held["a.weight_packing_meta"][1] == SCALE_LAYOUT_CODES["mma128"]
    assert torch.equal(meta, first)                                 # the checkpoint's own tensor is left as it was


def test_what_cannot_be_loaded_is_said():
    for held, rows, k, why in ((state("mma128", 128, 128, version=2)[0], 128, 128, "schema"),
                               (state("mma128", 128, 128, in_features=120)[0], 128, 128, "K = 120"),
                               (state("mma128", 128, 128)[0], 128, 160, "K = 128"),
                               (state("row_major", 128, 128)[0], 256, 128, "row_major"),
                               (state("mma64", 128, 128)[0], 128, 128, "mma64")):
        assert why in mxfp8_state_for_kernel(held, "a.", rows, k)
    assert mxfp8_state_for_kernel({}, "a.", 128, 128) is None        # nothing to load: strict loading says what is missing
    assert mxfp8_state_for_kernel({k: v.to("meta") for k, v in state("mma128", 128, 128)[0].items()}, "a.", 128, 128) is None
    held, _ = state("row_major", 128, 128)
    del held["a.weight_scales"]
    assert mxfp8_state_for_kernel(held, "a.", 128, 128) is None
