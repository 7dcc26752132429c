"""The prompt kernel's index arithmetic, read from its source on the CPU: what a row's registers
are indexed with stays within them for every width of a K/V tile."""
import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "kimi26-h100-rmsnorm-swiglu-fusion_b200", "csrc", "frn_prompt_attention.cu")


@pytest.mark.parametrize("keys", [96, 128])
def test_score_loads_stay_in_the_row(keys):
    """A row of scores has one register a key; loads of 32 columns must not go past the last."""
    with open(SOURCE) as f:
        text = f.read()
    assert re.search(r"float x\[kKeys\];", text) and f"{keys}" in text
    loops = re.findall(r"for \(int (\w+) = 0; \1 < ([^;]+); \+\+\1\)\s*\{?\s*tmem_ld_32x32b_x32\("
                       r"\w+ \+ \1 \* 32, reinterpret_cast<uint32_t\(&\)\[32\]>\(x\[\1 \* 32\]\)", text)
    assert loops, "no load of a row of scores was found"
    for _, bound in loops:
        count = eval(bound, {"kKeys": keys, "N": keys}) if "/" in bound else int(bound)
        assert count * 32 <= keys, f"{int(count)} loads of 32 columns into a row of {keys}"
