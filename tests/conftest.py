import os
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (REPO, os.path.join(REPO, "ml-cvnets_amd")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with `pytest -m gpu` on the GPU box)")


def pytest_collection_modifyitems(config, items):
    """`-m gpu` tests call the HIP library; skip them (not fail) when no GPU is visible so that a plain `pytest tests`
    on the CPU container stays green."""
    try:
        import torch
        has_gpu = torch.cuda.is_available()
    except Exception:  # pragma: no cover
        has_gpu = False
    if has_gpu:
        return
    skip = pytest.mark.skip(reason="no GPU visible")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


def _references_without_miopen():
    """The torch REFERENCE computations of the GPU tests (F.conv2d / batch_norm + autograd on the device) must not run MIOpen's solvers.
    Root cause of the asynchronous "Memory access fault by GPU" that rounds 3-4 saw in this suite: for the float32 1x1 convolution
    [2, 16, 6, 6] x [24, 16, 1, 1] of tests/test_kernels_gpu.py::test_bn_eval_mode, MIOpen's backward-data solver
    `igemm_bwd_gtcx35_nhwc_fp32_bx0_ex1_bt128x32x8_...` reads past the end of its operands.  Inside the caching allocator's segments that is
    invisible; when the tensor happens to end a segment that is followed by an unmapped range (allocation history = test order) the GPU
    faults.  Runs of that reference with torch alone (no kernel of this repository) under the guard-page allocator faulted with MIOpen and were clean
    without it (profiles/r05_fault_root_cause.txt); tools/guard_aten_repro.py makes the clean one only.  The product never calls MIOpen."""
    try:
        import torch
        torch.backends.cudnn.enabled = False  # ("cudnn" is MIOpen on ROCm): ATen's native convolution / batch-norm kernels instead
    except Exception:  # pragma: no cover
        pass


_references_without_miopen()


if os.environ.get("CVH_GUARD_ALLOC"):
    # debugging aid (tools/guard_alloc.cpp): every device allocation in its own address range with unmapped pages on both sides and never
    # reused after free — an out-of-bounds access or a launch through a stale pointer faults at the launch that does it
    import torch

    torch.cuda.memory.change_current_allocator(
        torch.cuda.memory.CUDAPluggableAllocator(os.path.abspath(os.environ["CVH_GUARD_ALLOC"]), "guard_malloc", "guard_free"))

    def _no_capture(*args, **kwargs):
        pytest.skip("no hipGraph capture under the guard allocator")

    torch.cuda.CUDAGraph = _no_capture


if os.environ.get("CVH_TEST_NAN_FILL"):
    # debugging aid: every torch.empty() buffer starts as NaN (floats) / max-int, so a kernel that reads memory it was supposed to
    # write first poisons the result deterministically instead of depending on what the caching allocator handed out
    import torch

    torch.use_deterministic_algorithms(True, warn_only=True)
    torch.utils.deterministic.fill_uninitialized_memory = True
