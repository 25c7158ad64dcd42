"""Which phases a loader has to wait for before its CTA leaves
(tinyoai_b200/csrc/ring.h), against a model of its rings: blocks of keys and of
values go through a ring each, and the loader may give up before any of them."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "tinyoai_b200" / "csrc"


@pytest.fixture(scope="module")
def last_parity(tmp_path_factory):
    d = tmp_path_factory.mktemp("ring")
    (d / "ring.cpp").write_text('#include "ring.h"\nextern "C" int last_parity(int sent, int stage, int stages) '
                                '{ return tcu::ring_last_parity(sent, stage, stages); }\n')
    subprocess.run(["g++", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(d / "ring.so"), str(d / "ring.cpp")], check=True)
    return C.CDLL(str(d / "ring.so")).last_parity


@pytest.mark.parametrize("stages", [1, 2, 3, 4])
def test_every_copy_is_waited_for(last_parity, stages):
    for blocks in range(1, 3 * stages + 2):
        for gave_up in range(2 * blocks + 1):  # keys and values of a block in turn, `gave_up` sent in all
            sent = [(gave_up + 1) // 2, gave_up // 2]
            for count in sent:
                # Copies of an earlier round on a stage have landed (that round's
                # release of the stage was waited for): the last of each stage are
                # what may be on its way, in the phase of its round.
                flying = {i % stages: i // stages for i in range(count)}
                for stage in range(stages):
                    want = flying[stage] & 1 if stage in flying else -1
                    assert last_parity(count, stage, stages) == want, (blocks, gave_up, count, stage)
