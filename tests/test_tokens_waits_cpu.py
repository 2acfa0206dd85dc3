"""The wait before a rescale in the prompt form of packed_attention, on a
model of its barriers: no GPU.

The MMA warp of a query tile issues, per key tile j, the products with V_j, the
scores of key tile j + 2 and the commits that announce them; commits arrive in
the order of issue, any time later.  A softmax warp that sees the scores of
key tile n may rescale O once the products with V_(n-1) are complete.  It
waits for that by the parity of a barrier's phase, which only tells
neighbouring phases apart.  The order of issue and the barriers are read from
the kernel's source.
"""
import re
from pathlib import Path

import pytest

SOURCE = Path(__file__).parent.parent / "uplift_b200" / "csrc" / "tok_attn_fwd.cu"
OLD = dict(order=("product", "scores", "o_done"), barriers=1)  # lets a wait pass a phase early


def of_source():
    text = SOURCE.read_text()
    loop = text[text.index("One tile's products at a time"):text.index("atomicExch(issuing, 0)")]
    at = {"product": loop.index("mma_tmem_a(o,"), "scores": loop.index("scores(ns + j + 2"),
          "o_done": loop.index("tc_commit(&o_done[")}
    commit = re.search(r"tc_commit\(&o_done\[(.*?)\]\)", loop).group(1)
    wait = re.search(r"wait\(&o_done\[(.*?)\], (.*?), 3\)", text).groups()
    barriers = {"t": 1, "2 * t + ((ns + j) & 1)": 2}[commit]
    assert wait == (("t", "(nn - 1) & 1") if barriers == 1 else ("2 * t + ((nn - 1) & 1)", "((nn - 1) >> 1) & 1"))
    return dict(order=tuple(sorted(at, key=at.get)), barriers=barriers)


def passes_early(order, barriers, tiles=9):
    """The first (n, arrivals so far) at which a wait for the products with V_(n-1) passes before they are complete."""
    events = [("scores", 0), ("scores", 1)]
    for j in range(tiles):
        events += [(what, j + 2 if what == "scores" else j) for what in order if what != "scores" or j + 2 < tiles]
    for n in range(1, tiles):
        for arrived in range(events.index(("scores", n)) + 1, len(events) + 1):
            past = events[:arrived]
            done = sum(what == "o_done" and j % barriers == (n - 1) % barriers for what, j in past)
            wanted = (n - 1) // barriers  # phase of the barrier; the wait passes if the one before the current has its parity
            if (done - 1) % 2 == wanted % 2 and ("o_done", n - 1) not in past:
                return n, past
    return None


def test_the_model_sees_an_early_wait():
    n, past = passes_early(**OLD)
    assert ("scores", n) in past and ("o_done", n - 2) not in past


def test_a_rescale_waits_for_the_last_product():
    assert passes_early(**of_source()) is None


@pytest.mark.parametrize("order,barriers", [(("product", "o_done", "scores"), 1), (("product", "scores", "o_done"), 2)])
def test_either_change_alone_would_do(order, barriers):
    assert passes_early(order, barriers) is None
