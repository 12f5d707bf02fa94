"""What the sources of attention over shared pages promise their callers, read from them (no GPU)."""
import os
import re

import pytest

from nnis_b200.csrc import build

FORMS = ["attention_shared.cu", "attention_shared_f32.cu", "attention_shared_mma.cu", "attention_shared_tc.cu", "attention_shared_warp.cu"]


@pytest.mark.parametrize("name", FORMS)
def test_positions_and_page_tables_are_read_behind_the_wait(name):
    """The kernel before a call may be the one that writes them: ahead of the wait for it a unit's kernel reads its plan alone."""
    with open(os.path.join(build.HERE, name)) as f:
        text = re.sub(r"//.*", "", f.read())
    begin = text.index("__launch_bounds__")  # (of the units' kernel, the file's first)
    ahead = text[begin:text.index("units_begin(a);", begin)]
    done = re.sub(r"auto \w+ = \[&\]\([^)]*\) \{.*?\n    \};|auto \w+ = \[&\].*?;\n", "", ahead, flags=re.S)  # (without what is only defined)
    assert not re.search(r"a\.token_pos\[|a\.page_table\[|\btable\[|\blook\(|a\.q\b|_cache\b", done), done
