"""A bounded wait whose outcome decides whether a warp goes on to instructions
that all its lanes have to meet (shuffles, votes, matrix and tensor-memory
instructions) has one outcome for the warp: each lane keeps its own time, so a
wait by lanes could end either way near its limit.  Read from the sources: a
wait that runs out cannot be made on a GPU on purpose.
"""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "tinyminigo_b200" / "csrc"

# the waits of whole warps that leave their loop when one gives up
WAITS = [
    ("attn_kv4.cu", r"full[warp][st], phase"),
    ("attn_tma.cu", r"full[s], ph)"),
    ("gemm_sm100.cu", r"acc_full[buf], (tl >> 1) & 1"),
    ("attn_prefill_tc.cu", r"o_full[bi], (i >> 1) & 1)) {"),
]


@pytest.mark.parametrize("name,barrier", WAITS)
def test_a_warps_wait_has_one_outcome(name, barrier):
    text = (CSRC / name).read_text()
    waits = [ln.strip() for ln in text.splitlines() if "mbar_wait" in ln and barrier in ln]
    assert len(waits) == 1, waits
    assert "mbar_wait_warp(" in waits[0], waits


def test_the_warps_wait_votes():
    text = (CSRC / "common.cuh").read_text()
    body = text[text.index("bool mbar_wait_warp("):]
    body = body[:body.index("\n}")]
    ends = re.findall(r"if \((.*)\) return (true|false);", body)
    assert [e for _, e in ends] == ["true", "false"]
    assert all(re.match(r"__(all|any)_sync\(0xffffffffu, ", c) for c, _ in ends), ends
