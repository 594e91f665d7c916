"""Guards on the GENERATED code of the persistent ping-pong kernels (CPU: disassembles the gfx950 code objects of the in-tree build).  The checks live in
scripts/codegen_guard.py, which the Makefile runs after every link (a failing guard or a missing llvm-objdump fails `make`, hence __graft_entry__.build()); this file holds the
same checks as tests.  Round 6: nothing skips any more - without an in-tree build the test BUILDS it (the driver runs build() first anyway)."""
import importlib.util
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_spec = importlib.util.spec_from_file_location("codegen_guard", os.path.join(ROOT, "scripts", "codegen_guard.py"))
guard = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(guard)


@pytest.fixture(scope="module")
def built():
    assert os.path.exists(guard.OBJDUMP), f"{guard.OBJDUMP} is missing: the code-generation guards cannot run"
    if not all(os.path.exists(os.path.join(guard.CSRC, o)) for o in list(guard.QUEUE_KERNELS) + list(guard.MARGIN_KERNELS)):
        subprocess.run(["make", "-C", guard.CSRC, "-j", "8", "GUARD=0"], check=True, capture_output=True)
    return True


@pytest.mark.parametrize("obj", sorted(guard.QUEUE_KERNELS))
def test_tile_queue_kernels_keep_the_ticket_register_and_use_no_scratch(obj, built):
    assert guard.check_object(obj) >= 2


@pytest.mark.parametrize("obj", sorted(guard.MARGIN_KERNELS))
def test_fp32_all_dma_kernels_keep_their_distance_between_a_barrier_and_the_next_lds_read(obj, built):
    assert guard.check_margins(obj) >= 2


@pytest.mark.parametrize("obj", sorted(guard.SEGMENT_KERNELS))
def test_token_product_has_a_segment_between_a_dmas_arrival_and_its_readers_barrier(obj, built):
    assert guard.check_segments(obj) >= 1


def test_a_wait_right_at_the_barrier_is_found():
    read, mma = ["ds_read_b128 v[0:3], v9"] * 12, ["v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]"] * 32
    wait, bar = ["s_waitcnt vmcnt(4)"], ["s_barrier"]
    assert guard.segment_waits(wait + read + bar + mma + bar + mma) == ["reads"]
    assert guard.segment_waits(read + wait + bar + mma + bar + mma) == ["mfmas"]
    assert guard.segment_waits(mma + wait + bar + read + bar + mma) == [None]
    assert guard.segment_waits(wait + ["s_sleep 4"] + bar + read + bar + mma) == ["sleep"]


def test_guard_script_exit_code(built):
    assert subprocess.run(["python3", os.path.join(ROOT, "scripts", "codegen_guard.py")], capture_output=True).returncode == 0
