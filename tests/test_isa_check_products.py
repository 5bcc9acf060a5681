"""The build's ISA check for loads into LDS through a buffer descriptor, and for matrix products
written in asm (both outside the compiler's own hazard recognizer)."""
import pytest

from block_lut_amd.csrc import isa_check as C
from test_isa_check import _text

LOAD = "buffer_load_dwordx4 v104, s[8:11], s0 offen lds"
PRODUCT = "v_mfma_f32_16x16x32_bf16 a[0:3], v[8:11], v[12:15], a[0:3]"


@pytest.mark.parametrize("lines, n", [
    (["v_readlane_b32 s11, v210, 46", LOAD], 1),                       # the descriptor's last word
    (["v_readlane_b32 s8, v210, 46", "s_nop 4", LOAD], 0),
    (["v_readfirstlane_b32 s0, v1", "s_nop 0", LOAD], 1),             # the offset
    (["v_readlane_b32 m0, v1, 2", "s_nop 3", LOAD], 1),
    (["v_readlane_b32 s12, v1, 2", LOAD], 0),
    (["v_readlane_b32 s11, v210, 46", "buffer_load_dwordx4 v[4:7], v104, s[8:11], s0 offen"], 0),   # the compiler's own
    (["v_mov_b32_e32 v9, v1", PRODUCT], 1),
    (["v_mov_b32_e32 v9, v1", "s_nop 1", PRODUCT], 0),
    (["v_accvgpr_write_b32 a3, 0", "s_nop 0", PRODUCT], 1),           # the addend
    (["v_permlane32_swap_b32_e32 v2, v12", PRODUCT], 1),              # (writes both)
    (["v_mov_b32_e32 v16, v9", PRODUCT], 0),
    ([PRODUCT, PRODUCT], 0),
])
def test_straight_line(lines, n):
    assert len(C.find_hazards(_text(lines))) == n
