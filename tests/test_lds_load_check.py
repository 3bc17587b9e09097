"""The build check of the inline-asm loads to LDS
(rust-deeplearning_amd/check_lds_loads.py): it passes on the compiled kernels
and fails on planted mistakes in small assembly fragments."""
import glob
import os
import re
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "rust-deeplearning_amd")
sys.path.insert(0, PKG)

import check_lds_loads as cl  # noqa: E402

LOAD = "buffer_load_dwordx4 v4, s[0:3], 0 offen lds"


def fn(*asm, before=(), after=(), name="_Z1kv"):
    return "\n".join([f"{name}:", *before, ";;#ASMSTART", *asm, ";;#ASMEND", *after, "s_endpgm", ".Lfunc_end0:"])


def test_compiled_kernels_hold():
    path = os.path.join(PKG, "build", "attention_batch.s")
    if not os.path.exists(path):
        pytest.skip("build/attention_batch.s is written by the library build (make -C rust-deeplearning_amd)")
    problems, checked = cl.check(open(path).read())
    assert checked > 0 and not problems, problems[:5]


def test_five_wait_states_pass():
    problems, checked = cl.check(fn("s_mov_b32 m0, s4", "s_nop 3", LOAD, before=["v_readfirstlane_b32 s0, v1"]))
    assert checked == 1 and not problems
    assert cl.check(fn("s_mov_b32 m0, s4", "s_nop 0x3", LOAD)) == ([], 1)


@pytest.mark.parametrize("nop", [[], ["s_nop 0"], ["s_nop 2"]])
def test_fewer_wait_states_fail(nop):
    # what stands before the block does not count: the compiler may move it
    problems, checked = cl.check(fn("s_mov_b32 m0, s4", *nop, LOAD, before=["s_nop 7"]))
    assert checked == 1 and problems and "wait states" in problems[0]


def test_a_load_without_its_address_fails():
    problems, _ = cl.check(fn("s_nop 4", LOAD))
    assert problems and "does not write M0" in problems[0]


def test_other_loads_are_not_checked():
    assert cl.check(fn("global_load_dwordx4 v[4:7], v[2:3], off")) == ([], 0)


def test_m0_read_behind_a_block_fails():
    asm = ["s_mov_b32 m0, s4", "s_nop 3", LOAD]
    problems, _ = cl.check(fn(*asm, before=["s_mov_b32 m0, s9"], after=["v_movrels_b32 v1, v2, m0"]))
    assert problems and "M0 read" in problems[0]
    assert cl.check(fn(*asm, after=["s_mov_b32 m0, s9", "s_add_u32 s1, m0, s2"])) == ([], 1)
    assert cl.check(fn(*asm, after=["s_add_u32 m0, m0, s2"]))[0]


def test_blocks_that_write_m0_say_so():
    # the compiler may keep a value there over a block that does not name it
    blocks = []
    for path in glob.glob(os.path.join(PKG, "csrc", "*.h*")):
        blocks += re.findall(r"\basm\b[^;]*?\)\s*;", open(path).read())
    writers = [b for b in blocks if re.search(r"\bm0\s*,", b)]
    assert len(blocks) > 5 and writers
    for b in writers:
        assert '"m0"' in b.rsplit(":", 1)[1], b
