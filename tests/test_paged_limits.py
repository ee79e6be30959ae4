"""Sizes at which the counts of a plan of the attention over a paged cache end."""
import os
import subprocess
import sys

import pytest

from archscale_b200.ops import backend

pytestmark = pytest.mark.skipif(backend.extension_path() is None, reason="the extension is not built")


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("B,T,H,G,D", [(1, 1 << 30, 4, 1, 4), (2, 1 << 30, 8, 2, 64), (1, (1 << 31) - 1, 1, 1, 128), (1, (1 << 31) - 1, 3, 1, 64), (1, 1 << 29, 64, 16, 128)])
def test_more_query_rows_of_a_key_head_than_32_bits_count(B, T, H, G, D, e4m3):
    """They are left to the kernel of one query row per CTA, which refuses what its grid does not hold; in a process of its own, which a division by zero would end."""
    code = f"import paged_plan; assert paged_plan.workspace({B}, {T}, {H}, {G}, {D}, 64, 100, e4m3={e4m3}) == 0"
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join((here, os.path.dirname(here))))
    done = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
