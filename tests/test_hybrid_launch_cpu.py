"""Launch plans of the hybrid family's kernels ask how many SMs there are."""
import pathlib
import re

CSRC = pathlib.Path(__file__).resolve().parents[1] / "llaminar_b200" / "ops" / "csrc"


def test_no_plan_has_a_number_of_sms():
    for name in ("gdn_rows.cu", "gdn_chunk.cu", "rope_part.cu", "attn_shared.cu"):
        code = "\n".join(line.split("//")[0] for line in (CSRC / name).read_text().splitlines())
        assert not re.search(r"\b148\b", code) and "sm_count()" in code, name
