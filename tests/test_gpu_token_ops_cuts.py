"""gated_recurrence over histories that are cut into several pieces of several tiles each, with memories that
span the pieces, against the 64-bit definition."""
import pytest
import torch

from test_gpu_token_ops import DEV, IDS, DTYPES, check_recurrence, gen_of, rnd
from token_cuts import CUT_SHAPES

pytestmark = pytest.mark.gpu


def remembering_case(b, t, d, dtype, logits, key, resets, lengths):
    """Memories of about 2000 steps, and a few resets among them."""
    gen = gen_of(b, t, d, key)
    g = 7.0 + torch.randn(b, t, d, generator=gen) if logits else 1.0 - 0.001 * torch.rand(b, t, d, generator=gen)
    return {"x": rnd(gen, b, t, d, dtype=dtype), "g": g.to(DEV), "h0": rnd(gen, b, d) * 30.0,
            "resets": (torch.rand(b, t, generator=gen) < 3.0 / t).to(DEV) if resets else None,
            "lengths": (t - torch.randint(0, t // 2, (b,), generator=gen)).to(DEV) if lengths else None,
            "d_h": rnd(gen, b, t, d, dtype=dtype), "d_last": rnd(gen, b, d) * 30.0}


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("logits", [True, False], ids=["logit", "decay"])
@pytest.mark.parametrize("b,t,d", CUT_SHAPES)
def test_gated_recurrence_cut_into_pieces_of_several_tiles(b, t, d, logits, dtype):
    for key, (reverse, resets, lengths) in enumerate([(False, False, False), (True, True, b > 1)]):
        c = remembering_case(b, t, d, dtype, logits, key, resets, lengths)
        check_recurrence(c, logits, reverse, dtype, torch.float32, f"reverse {reverse}: ")
