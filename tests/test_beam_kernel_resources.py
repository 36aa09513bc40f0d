"""What beam search's kernels hold on a compute unit (see test_kernel_resources.py)."""
import re

import pytest

from deliverance_amd.kernels import build
from test_kernel_resources import LANES, LDS, REGISTERS, _code_objects, _notes


def kernels(unit, name):
    """Template arguments as they stand in the symbol -> (workgroups a compute unit, scratch bytes a lane)."""
    try:
        build.build(only=[unit], verbose=False)
    except build.KernelLibraryError as e:
        pytest.skip(str(e))
    with open(build.unit_path(unit), "rb") as f:
        blob = f.read()
    found = {}
    for elf in _code_objects(blob):
        for k in _notes(elf):
            m = re.match(r"_Z\d+%s(?:I([a-z]?)((?:Li\d+E)+)E)?" % name, k[".name"])
            if m:
                waves = -(-k[".max_flat_workgroup_size"] // LANES)
                a_simd = min(8, REGISTERS // (-(-max(1, k[".vgpr_count"]) // 8) * 8))
                fit = min(4 * a_simd // waves, LDS // max(1, k[".group_segment_fixed_size"]))
                found[(m[1], *(int(x) for x in re.findall(r"Li(\d+)E", m[2] or "")))] = (fit, k[".private_segment_fixed_size"])
    assert found, f"{name} is not in {unit}"
    return found


def test_attention_of_beams_does_not_spill():
    """No scratch memory; 8 wavefronts of head sizes up to 128 fill a compute unit, 4 of them leave room for a second workgroup; every form
    that is compiled is one that a call asks for."""
    found = kernels("attn_beams", "attn_beams_kernel")
    for (kind, dk, step, waves, tiles), (workgroups, scratch) in found.items():
        assert scratch == 0, (kind, dk, step, waves, tiles)
        assert workgroups >= (2 if waves == 4 and dk <= 4 else 1), (kind, dk, step, waves, tiles)
    forms = {(1, 8, 1), (1, 4, 1), (1, 8, 2), (2, 8, 1), (2, 4, 1), (2, 8, 2), (4, 8, 1), (4, 4, 1), (8, 4, 1)}
    assert {(kind, dk, waves, tiles) for kind, dk, _, waves, tiles in found} == {(kind, *f) for kind in "ft" for f in forms}


@pytest.mark.parametrize("unit,name", [("beam_select", "beam_stats_kernel"), ("beam_select", "beam_choose_kernel"), ("attn_beams", "attn_beams_merge_kernel")])
def test_the_others_do_not_spill(unit, name):
    try:
        found = kernels(unit, name)
    except AssertionError:
        pytest.fail(f"{name} is not in {unit}")
    assert all(scratch == 0 and workgroups >= 1 for workgroups, scratch in found.values())


def test_reordering_does_not_spill():
    """A thread of the widest form keeps 64 columns; every form is compiled and has no scratch memory."""
    try:
        build.build(only=["reorder"], verbose=False)
    except build.KernelLibraryError as e:
        pytest.skip(str(e))
    with open(build.unit_path("reorder"), "rb") as f:
        found = {k[".name"]: k[".private_segment_fixed_size"] for elf in _code_objects(f.read()) for k in _notes(elf) if "reorder_kernel" in k[".name"]}
    assert len(found) == 5 and not any(found.values()), found
