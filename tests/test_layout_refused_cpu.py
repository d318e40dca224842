"""The lane-per-env layout (envs_per_block > 0) is refused before anything touches a GPU; a run of it was aborted because its
scratch could not be allocated, and the cause is not known."""
import ctypes

import pytest

from ur3e_amd import runtime as rt


@pytest.mark.parametrize("epb", [1, 16, 64, 65])
@pytest.mark.parametrize("task", [rt.TASK_GYM_V2, rt.TASK_GYM_V0])
def test_one_env_a_lane_is_refused(epb, task):
    md, mc = rt.load_model("main")
    cfg = rt.make_config(task=task, frame_skip=2, model=md, envs_per_block=epb)
    L = rt.load_library()
    h = ctypes.c_void_p()
    assert L.ur3e_batch_create(ctypes.byref(mc), ctypes.byref(cfg), 64, 0, ctypes.byref(h)) == -1  # UR3E_EINVAL
    assert b"one env per lane" in L.ur3e_last_error() and not h.value
