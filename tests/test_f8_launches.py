"""Whether a launch may overlap the one before it is for the runtime to say, in the newer sources too."""
from __future__ import annotations

import pytest

from vinf_3080ti_b200 import build


@pytest.mark.parametrize("name", ["vqm_qmm_f8.cu", "vqm_rows_f8.cu", "vqm_logprobs.cu"])
def test_no_launcher_asks_for_overlap_by_itself(name):
    source = (build.CSRC / name).read_text()
    assert "launch_attributes(" in source and "ProgrammaticStreamSerialization" not in source
