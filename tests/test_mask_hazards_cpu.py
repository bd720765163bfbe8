"""Masks that inline asm takes from comparisons (the counts of klp_top.hip) keep
the two wait states between a vector write of an SGPR and a vector read of it
(the generated assembly, checked by tests/mfma_hazards.py)."""
from __future__ import annotations

import re

import pytest

import isa_listing
from mfma_hazards import hazards, hazards_of_kernel

READERS = [("v_cmp_ge_f32_e32 vcc, v1, v2", "v_addc_co_u32_e32 v3, vcc, 0, v3, vcc"),
           ("v_cmp_ge_f32_e32 vcc, v1, v2", "v_cndmask_b32_e32 v3, v4, v5, vcc"),
           ("v_cmp_ge_f32_e64 s[4:5], v1, v2", "v_addc_co_u32_e64 v3, vcc, 0, v3, s[4:5]"),
           ("v_add_co_u32_e32 v3, vcc, v1, v2", "v_addc_co_u32_e32 v4, vcc, 0, v4, vcc"),
           ("v_readfirstlane_b32 s6, v1", "v_add_f32_e32 v3, s6, v3")]


@pytest.mark.parametrize("writer,reader", READERS)
def test_detector_counts_wait_states(writer, reader):
    for n in range(4):
        body = ["; %bb.0:", "\t" + writer] + ["\tv_mov_b32_e32 v20, 0"] * n
        found = hazards_of_kernel(body + ["\t" + reader, "\ts_endpgm"])
        assert bool(found) == (n < 2), (n, found)
    assert not hazards_of_kernel(["; %bb.0:", "\t" + writer, "\ts_nop 1", "\t" + reader,
                                  "\ts_endpgm"])


def test_detector_leaves_results_and_branches():
    # A carry written again, a branch, another register.
    for reader in ("v_add_co_u32_e32 v3, vcc, v1, v2", "v_cmp_lt_f32_e32 vcc, v1, v2",
                   "s_cbranch_vccz .LBB0_1", "v_cndmask_b32_e64 v3, v4, v5, s[8:9]"):
        body = ["; %bb.0:", "\tv_cmp_ge_f32_e32 vcc, v1, v2", "\t" + reader, ".LBB0_1:",
                "\ts_endpgm"]
        assert hazards_of_kernel(body) == []


@pytest.mark.skipif(not isa_listing.available(), reason="hipcc not available")
def test_counts_have_wait_states():
    listing = isa_listing.listing("klp_top.hip")
    blocks = re.findall(r";;#ASMSTART\n(.*?);;#ASMEND", listing, re.S)
    assert any("v_addc_co_u32" in b for b in blocks)
    found = hazards(listing)
    assert not found, {k: (len(v), v[:2]) for k, v in found.items()}
