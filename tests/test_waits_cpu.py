"""Every wait in a kernel gives up after a while and says so.  A kernel that does not look at the answer goes on with
data that has not arrived, and waits again for each piece that follows: a result that is dropped has to be dropped
on purpose, by a (void) or with the reason behind it."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "turt_b200" / "csrc"


@pytest.mark.parametrize("path", sorted(CSRC.glob("*.cu*")), ids=lambda p: p.name)
def test_no_wait_is_ignored(path):
    dropped = [f"{i}: {line.strip()}" for i, line in enumerate(path.read_text().splitlines(), 1)
               if re.match(r"\s*mbar_wait\w*\(", line) and "//" not in line]
    assert not dropped
