"""Filtered sampling where a row's mass is spread over millions of tokens: flat rows of the largest
vocabulary, and tails whose tokens weigh less than 2^-43 of the largest each."""
import numpy as np
import pytest
import torch

from gpu_util import say
from test_gpu_paged_serving import sample

pytestmark = pytest.mark.gpu
MOST = 2**21
ENDS = [0.0, 0.06, 0.1219, 0.1222, 0.1245, 0.1249, 0.125, 0.2, 0.2495, 0.3, 0.3749, 0.4, 0.4999, 0.5,
        0.55, 0.6249, 0.7, 0.7499, 0.8, 0.8749, 0.9, 0.9749, 0.9765, 0.99, 0.9995, 0.99999, 1 - 2**-22,
        1 - 2**-24, 1.0, 2.0, float("inf"), 0.997, 0.11]


def flat_tokens(kept):
    """The first `kept` ids weigh the same: floor(u x kept), the last one for u >= 1."""
    return [min(int(float(np.float32(min(x, 1.0))) * kept), kept - 1) for x in ENDS]


@pytest.mark.parametrize("vocab", [2046403, MOST])
@pytest.mark.parametrize("how", ["off", "hot", "min_p", "top_p"])
def test_flat_rows_of_the_largest_vocabulary(hip, ctx, vocab, how):
    """Every token of a chunk can be drawn, its last ones too: rows of equal weights, cut into 8 chunks
    (33 rows), at draws on both sides of the chunks' ends.  The weights are 1 and the products u x kept
    exact, so that the tokens are floor(u x kept)."""
    say(f"sample: flat rows of {vocab}, {how}")
    rows = len(ENDS)
    assert rows == 33
    kept, t, p, m = vocab, None, None, None
    if how == "hot":                        # any finite logits weigh the same
        logits = torch.empty(rows, vocab, device="cuda").normal_(
            0.0, 2.0, generator=torch.Generator(device="cuda").manual_seed(5))
        t = [float("inf")] * rows
    else:
        logits = torch.full((rows, vocab), 2.5, device="cuda")
    if how == "min_p":
        m = [0.5] * rows
    if how == "top_p":
        kept, p = -(-3 * vocab // 4), [0.75] * rows
    got = sample(hip, ctx, logits, t, None, p, m, ENDS)
    want = flat_tokens(kept)
    assert got == want, [(u, g, w) for u, g, w in zip(ENDS, got, want) if g != w][:8]


def test_top_k_holds_among_tokens_that_weigh_next_to_nothing(hip, ctx):
    """One token, 2^20 of 2^-43.2 of its weight and as many of 2^-45; top_k ends among the last ones, top_p
    before them.  A uniform of zero draws the first kept id: the large token (the others may count as
    nothing) or one that both filters keep, never one of the last."""
    say("sample: top-k and top-p among tokens of next to no weight")
    logits = torch.full((2, MOST), -29.95, device="cuda")
    logits[:, MOST // 2:] = -31.2
    logits[:, MOST - 1] = 0.0
    w = np.exp(np.float64(np.float32(-29.95)))
    top_p = 1 - 2**-24
    n_light = int(np.ceil((top_p * (1 + w * 2**20) - 1) / w))     # of the 2^20, those within top_p
    assert 0 < n_light < 2**20
    for k, p in ((2**20 + 1001, top_p), (0, top_p)):
        got = sample(hip, ctx, logits, None, [k] * 2, [p] * 2, None, [0.0, 0.5])
        assert got[0] < n_light or got[0] == MOST - 1, (k, p, got)
        assert got[1] == MOST - 1
