"""Binding an 8-bit tensor while a graph is captured: a new name is only noted; to replace a tensor means to wait and to free, which a capture does not
bear, so it is refused and the capture goes on."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_replacing_a_tensor_beside_a_capture_is_refused():
    import torch

    from vinf_3080ti_b200.runtime import Runtime

    rt = Runtime()
    w, s = torch.ones((4, 48), dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    torch.cuda.synchronize()
    rt.upload_i8("mine", np.full((4, 48), 2, np.int8), np.ones(4, np.float32), 48, 4)
    rt.bind_i8("bound", w.data_ptr(), s.data_ptr(), 48, 4)
    for name, n, elem in (("q", 48, 1), ("s", 1, 4), ("y", 4, 4), ("y2", 4, 4)):
        rt.alloc(name, n, elem)
    rt.write("q", np.ones(48, np.int8))
    rt.write("s", np.ones(1, np.float32))
    rt.capture_begin()
    rt.qmm_i8("mine", "q", "s", "y")
    for name in ("mine", "bound"):
        with pytest.raises(ValueError, match="captured"):
            rt.bind_i8(name, w.data_ptr(), s.data_ptr(), 48, 4)
    rt.bind_i8("new", w.data_ptr(), s.data_ptr(), 48, 4)
    rt.qmm_i8("new", "q", "s", "y2")
    graph = rt.capture_end()
    rt.graph_launch(graph)
    assert rt.read_array("y").tolist() == [96.0] * 4 and rt.read_array("y2").tolist() == [48.0] * 4
    rt.bind_i8("bound", w.data_ptr(), s.data_ptr(), 48, 3)  # afterwards it may be replaced
    assert rt.tensor_info("bound")[2:4] == (3, 48)
    rt.graph_destroy(graph)
    rt.close()
