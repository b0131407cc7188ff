"""A further wait state that gfx950 needs from the program, checked in the listing of every kernel of the built library: a
v_readlane / v_readfirstlane reads a vector register at least one wait state behind the vector instruction that wrote it, and
a vector instruction reads a scalar register at least two behind the vector instruction that wrote it (around inline asm the
compiler puts none)."""
import re

from test_wait_states import _insns, _sgprs, _vregs, _within, kernels  # noqa: F401


def readlane_gaps(insns):
    """The lane reads right behind the vector instruction that wrote the register they read."""
    reads = {i: _vregs(args.split(", ")[1]) for i, (op, args, _) in enumerate(insns)
             if op.startswith(("v_readlane", "v_readfirstlane"))}
    return [j for i, (op, args, _) in enumerate(insns)
            if reads and op.startswith("v_") and not op.startswith(("v_cmp", "v_readlane", "v_readfirstlane", "v_mfma"))
            for j in _within(insns, i, 1) if j in reads and _vregs(args.split(", ")[0]) & reads[j]]


def scalar_gaps(insns):
    """The vector instructions fewer than two wait states behind the lane read that wrote a scalar register of theirs."""
    out = []
    for i, (op, args, _) in enumerate(insns):
        if op.startswith(("v_readlane", "v_readfirstlane")):
            dest = _sgprs(args.split(", ")[0])
            out += [j for j in _within(insns, i, 2) if insns[j][0].startswith("v_")
                    and _sgprs(", ".join(insns[j][1].split(", ")[1:])) & dest]
    return out


def test_lane_reads_are_late_enough(kernels):  # noqa: F811
    bad = {k: len(g) for k, g in ((k, readlane_gaps(ins)) for k, ins in kernels.items()) if g}
    assert not bad, bad


def test_scalars_from_lanes_are_read_late_enough(kernels):  # noqa: F811
    bad = {k: len(g) for k, g in ((k, scalar_gaps(ins)) for k, ins in kernels.items()) if g}
    assert not bad, bad


def test_the_checks():
    write, read = "v_mov_b32_e32 v6, s74", "v_readfirstlane_b32 s79, v6"
    assert readlane_gaps(_insns(write, read)) == [1] and readlane_gaps(_insns(write, "s_nop 0", read)) == []
    assert readlane_gaps(_insns(write, "v_readfirstlane_b32 s79, v7")) == []
    use = "v_add_u32_e32 v1, s79, v2"
    assert scalar_gaps(_insns(read, "s_nop 0", use)) == [2] and scalar_gaps(_insns(read, "s_nop 1", use)) == []
    assert not re.search("s79", write)
