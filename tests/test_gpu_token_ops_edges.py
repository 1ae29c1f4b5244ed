"""The token-policy operators on the GPU at the edges of what their interfaces allow.  Definitions and
bounds: tests/token_oracle.py."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import token_oracle as O
from test_gpu_token_ops import DEV, DTYPES, IDS, check_log_probs, gen_of, np64, rnd

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------- states written in place
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("b,d", [(1, 1), (3, 33), (200, 65), (5, 64), (70, 1025)])
def test_single_step_that_keeps_states_and_writes_them_in_place(dtype, b, d):
    """pa_gated_recurrence with T = 1, `last` = h0 and `carries`: every channel's old state is read, and kept
    for the gradient, before the new one is written, also where a row's last channels share a pack."""
    from pearl_amd import _native as N, gated_recurrence_grad
    gen = gen_of(b, d, 91)
    x, g, h0 = rnd(gen, b, 1, d, dtype=dtype), rnd(gen, b, 1, d, dtype=dtype), rnd(gen, b, d)
    d_h, d_last = rnd(gen, b, 1, d, dtype=dtype), rnd(gen, b, d)
    want = O.recurrence(np64(x), np64(g), np64(h0), None, None, True, False, np64(d_h), np64(d_last))
    code = {torch.float32: N.PA_F32, torch.bfloat16: N.PA_BF16, torch.float16: N.PA_F16}[dtype]
    assert N.lib().pa_gated_recurrence_carries(b, 1, d) == b * d
    for _ in range(5):
        state, kept, h = h0.clone(), torch.full((b * d,), float("nan"), device=DEV), torch.empty_like(x)
        args = N.RECURRENCE_ARGS.pack(0, code, code, 1, 0, d, b, 1, x.data_ptr(), d, 0, g.data_ptr(), d, 0, state.data_ptr(),
                                      0, 0, 0, 0, h.data_ptr(), state.data_ptr(), kept.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0)
        N.check(N.lib().pa_gated_recurrence(args, N.stream_ptr(x.device)))
        assert torch.equal(kept.view(b, d), h0)
        O.check(h, *want["h"], dtype, "h")
        O.check(state, *want["last"], torch.float32, "last")
    dx, dg, d0 = gated_recurrence_grad(x, g, kept, d_h, d_last)
    for got, name, kind in ((dx, "d_x", dtype), (dg, "d_g", dtype), (d0, "d_h0", torch.float32)):
        O.check(got, *want[name], kind, name)


# ---------------------------------------------------------------------------- tangents
def test_tangents_are_refused_and_plain_calls_beside_them_run():
    from pearl_amd import action_log_probs, embed_tokens, gated_recurrence, gated_recurrence_step
    x, tok = torch.randn(3, 4, 8, device=DEV), torch.tensor([[0, 1], [2, 2]], device=DEV)
    w, act = torch.randn(3, 8, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    want = embed_tokens(w, tok)
    with forward_ad.dual_level():
        dual, wide = forward_ad.make_dual(w, torch.ones_like(w)), forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: embed_tokens(dual, tok), lambda: gated_recurrence(wide, x), lambda: gated_recurrence(x, wide),
                     lambda: gated_recurrence(x, x, forward_ad.make_dual(x[:, 0], x[:, 1])),
                     lambda: gated_recurrence_step(dual, w), lambda: action_log_probs(dual, act),
                     lambda: gated_recurrence(wide.requires_grad_(), x)):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(embed_tokens(w, tok), want)


# ---------------------------------------------------------------------------- log probabilities
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("width", [10, 400, 9000])
def test_action_log_probs_at_the_largest_and_smallest_temperature(dtype, width):
    gen = gen_of(width, 81)
    logits = rnd(gen, 6, width, dtype=dtype, scale=2.0)
    mask = (torch.rand(6, width, generator=gen) < 0.4).to(DEV)
    mask[:, 1] = False
    logits[2, 2] = float("-inf")
    logits[3, 3:] = torch.finfo(dtype).min
    logits[4, 1] = torch.finfo(dtype).max
    actions = torch.ones(6, dtype=torch.int64, device=DEV)
    g_lp, g_h = rnd(gen, 6), rnd(gen, 6)
    for temperature in (2.0 ** 121, 2.0 ** 60):
        check_log_probs(logits, actions, mask, temperature, 4, dtype, g_lp, g_h, f"T {temperature}: ")
        check_log_probs(logits, actions, None, temperature, 0, dtype, g_lp, None, f"T {temperature}, no mask: ")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("width", [10, 400, 9000])
def test_action_log_probs_infinite_gradients_stay_away_from_unavailable_actions(dtype, width):
    from pearl_amd import action_log_probs, action_log_probs_grad
    inf = float("inf")
    gen = gen_of(width, 83)
    logits = rnd(gen, 6, width, dtype=dtype, scale=2.0)
    mask = (torch.rand(6, width, generator=gen) < 0.4).to(DEV)
    mask[:, 2] = False
    logits[:, 7] = float("-inf")
    off = mask | (logits == float("-inf"))
    actions = torch.full((6,), 2, device=DEV)
    g_lp, g_h = rnd(gen, 6), rnd(gen, 6)
    o = action_log_probs(logits, actions, mask)
    plain = action_log_probs_grad(o, logits, actions, g_lp, g_h, mask)
    g_lp[0], g_h[1], g_lp[2], g_h[3] = inf, inf, -inf, float("nan")
    for some in ((g_lp, g_h), (g_lp, None), (None, g_h)):
        d = action_log_probs_grad(o, logits, actions, *some, mask)
        assert (d[off] == 0).all()
        assert torch.isfinite(d[4:]).all()
    d = action_log_probs_grad(o, logits, actions, g_lp, g_h, mask)
    assert torch.equal(d[4:], plain[4:])
    on = ~off
    on[:, 2] = False
    assert (d[0][on[0]] == -inf).all() and (d[2][on[2]] == inf).all() and torch.isnan(d[3][on[3]]).all()


@pytest.mark.parametrize("width", [10, 400, 9000])
def test_action_log_probs_gradients_that_overflow_leave_the_others_alone(width):
    """g / T passes the range of a float: where p or 1 - p is zero the gradient is zero all the same."""
    from pearl_amd import action_log_probs, action_log_probs_grad
    logits = -torch.arange(width, device=DEV, dtype=torch.float32).repeat(2, 1) - 1.0
    actions = torch.tensor([0, 1], device=DEV)
    o = action_log_probs(logits, actions, temperature=2.0e-38)      # distances of 5e37 and more: p is 1, 0, 0, ...
    d = action_log_probs_grad(o, logits, actions, torch.full((2,), 10.0, device=DEV), temperature=2.0e-38)
    want = torch.zeros(2, width, device=DEV)
    want[1, 0], want[1, 1] = float("-inf"), float("inf")
    assert torch.equal(d, want)


def test_action_log_probs_the_largest_entropy_gradients():
    """g_H (log p + H) passes the range of a float for every p that has underflowed, and only there counts for nothing."""
    from pearl_amd import action_log_probs, action_log_probs_grad
    for width in (10, 400, 9000):
        logits = torch.full((2, width), -1000.0, device=DEV)
        logits[:, 0] = 0.0
        logits[:, 1] = float("-inf")
        actions = torch.zeros(2, dtype=torch.int64, device=DEV)
        o = action_log_probs(logits, actions)
        for g in (3.0e38, 1.0e35):
            d = action_log_probs_grad(o, logits, actions, None, torch.full((2,), g, device=DEV))
            assert (d == 0).all(), (width, g)


@pytest.mark.parametrize("width", [10, 400, 20000])
def test_action_log_probs_of_logits_further_apart_than_a_float_holds(width):
    gen = gen_of(width, 82)
    for dtype in (torch.float32, torch.bfloat16):
        logits = rnd(gen, 4, width, dtype=dtype)
        logits[:, 0] = 3.2e38
        logits[1, 1:] = -3.2e38
        logits[2, 5] = -3.0e38
        actions = torch.tensor([0, 3, 5, 5], device=DEV)
        check_log_probs(logits, actions, None, 16.0, 4, dtype, rnd(gen, 4), rnd(gen, 4), "far: ")


def test_a_state_written_in_place_is_known_to_autograd():
    from pearl_amd import gated_recurrence_step
    x, g, state = (torch.randn(3, 8, device=DEV) for _ in range(3))
    w = torch.ones(8, device=DEV, requires_grad=True)
    y = (state * w).sum()                                     # keeps the state for w's gradient
    gated_recurrence_step(x, g, state, out_state=state)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    with torch.inference_mode():
        kept = torch.zeros(3, 8, device=DEV)
    for _ in range(2):
        gated_recurrence_step(x, g, kept, out_state=kept)      # made in inference mode: nothing to tell
    leaf = torch.zeros(3, 8, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError):
        gated_recurrence_step(x, g, out_state=leaf)
