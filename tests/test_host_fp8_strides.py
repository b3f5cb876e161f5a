"""Strides and lengths that would wrap in 64 bits are refused, without a GPU: the C entry points check
before any launch."""

from __future__ import annotations

import pytest

A, B, C, D = 0x10000, 0x40000000, 0x80000000, 0xC0000000  # addresses that are never followed


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("ld", [2**62, 2**63 - 64, 2**61, 2**22 + 16])
def test_linear_refuses_strides_that_wrap(pkg, dtype, ld):
    lib = pkg._lib.load()
    scale = D if dtype else None
    for ldx, ldw in ((ld, 64), (64, ld)):
        assert lib.moe_linear(A, ldx, scale, B, ldw, scale, dtype, 4, 64, 8, None, 0, 0, None, None, C,
                              None) == pkg._lib.MOE_EINVAL
        assert b"ldx and ldw" in lib.moe_last_error()


def test_experts_fp8_gate_logits_keep_clear_of_the_outputs(pkg):
    """The shared gate's logits, one of `ld` bf16, are an input as the others; their stride may not wrap."""
    lib = pkg._lib.load()
    need = lib.moe_experts_fp8_workspace_bytes(4, 64, 8, 2, 32)

    def call(gate, ld):
        return lib.moe_experts_fp8_forward(A, B, 4, 64, 8, 2, 32, B, B, B, B, B, B, B, gate, ld, None, C, D, need, None)

    for gate, ld, words in ((C, 1, b"overlap"), (C + 510, 1, b"overlap"), (C - 6 * 40, 40, b"overlap"),
                            (D + 64, 3, b"overlap"), (B, 2**31, b"gate"), (B, 2**62, b"gate"), (B, -1, b"gate")):
        assert call(gate, ld) == pkg._lib.MOE_EINVAL, (gate, ld)
        assert words in lib.moe_last_error()
