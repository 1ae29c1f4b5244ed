"""The token-policy operators on the GPU at the edges of what their interfaces allow.  Definitions and
bounds: tests/token_oracle.py."""
import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import token_oracle as O
from test_gpu_token_ops import DEV, DTYPES, IDS, check_log_probs, check_recurrence, gen_of, np64, rnd

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


# ---------------------------------------------------------------------------- decays above one
def growing_case(b, t, d, dtype, gate_dtype, key, resets=False, lengths=False):
    """Channels whose products of decays leave the range of a float while their states stay inside it.
    Kind 0: nothing but zeros meets growth.  1: zeros grow, then a decay of zero, then an ordinary history.
    2: a state of 1e-30 grows by 1e50 and shrinks again.  3: factors of 1e10 and 1e-10 in turn.  4: ordinary."""
    gen = gen_of(b, t, d, key)
    half = t // 2
    grow = 10.0 ** (50.0 / half) if half else 1.5
    x, d_h = torch.randn(b, t, d, generator=gen), torch.randn(b, t, d, generator=gen)
    g = 0.7 + 0.3 * torch.rand(b, t, d, generator=gen)
    h0, d_last = torch.randn(b, d, generator=gen), torch.randn(b, d, generator=gen)
    for c in range(d):
        kind = (c + key) % 5
        if kind == 0:
            g[:, :, c], x[:, :, c], h0[:, c], d_h[:, :, c], d_last[:, c] = 1.5 * grow, 0.0, 0.0, 0.0, 0.0
        if kind == 1:
            g[:, :half, c], x[:, :half, c], h0[:, c] = grow * grow, 0.0, 0.0
            g[:, half, c] = 0.0
            d_h[:, :half, c] = 0.0
        if kind == 2:
            g[:, :half, c], g[:, half:, c] = grow, 1.0 / grow
            x[:, :, c] = 0.0
            h0[:, c] *= 1e-30
            d_h[:, :, c] *= 1e-30
            d_last[:, c] *= 1e-30
        if kind == 3:
            g[:, 0::2, c], g[:, 1::2, c] = 1e10, 1e-10
    case = {"x": x.to(dtype), "g": g.to(gate_dtype), "h0": h0, "d_h": d_h.to(dtype), "d_last": d_last,
            "resets": torch.rand(b, t, generator=gen) < 3.0 / t if resets else None,
            "lengths": torch.randint(0, t + 1, (b,), generator=gen) if lengths else None}
    return {k: None if v is None else v.to(DEV) for k, v in case.items()}


# one step; one wave; one tile of half-width slabs; one tile and a cut of one tile a chunk; several tiles a
# chunk; histories that are not cut; and a last slab of three channels after one of two fewer
@pytest.mark.parametrize("b,t,d", [(2, 1, 10), (2, 24, 10), (1, 32, 37), (2, 100, 10), (1, 230, 10), (1, 2000, 10),
                                   (26, 1300, 10), (140, 600, 5), (2, 24, 33), (2, 100, 65), (3, 300, 65), (1, 1500, 129)])
@pytest.mark.parametrize("dtype,gate_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                              (torch.bfloat16, torch.bfloat16)], ids=["fp32", "bf16-fp32", "bf16"])
def test_gated_recurrence_decays_above_one(b, t, d, dtype, gate_dtype):
    with np.errstate(all="ignore"):
        for key, (reverse, resets, lengths) in enumerate([(False, False, False), (True, True, True)]):
            c = growing_case(b, t, d, dtype, gate_dtype, key, resets, lengths)
            if reverse:
                c["g"], c["x"], c["d_h"] = (c[k].flip(1).contiguous() for k in ("g", "x", "d_h"))
            check_recurrence(c, False, reverse, dtype, gate_dtype, f"reverse {reverse}: ")


def test_gated_recurrence_decays_above_one_leave_equal_bits():
    """Channels beside those that grow, in the same workgroup and in the next: the same bits every time."""
    from pearl_amd import gated_recurrence, gated_recurrence_grad
    for t, d in ((24, 33), (100, 65), (1500, 129)):
        gen = gen_of(t, d, 95)
        x, d_h = rnd(gen, 2, t, d), rnd(gen, 2, t, d)
        for at in (0, d - 10, d - 2, d - 1):
            g = (0.9 + 0.05 * torch.rand(2, t, d, generator=gen)).to(DEV)
            g[0, t // 3, at] = 1.5
            first = None
            for _ in range(6):
                h, last, kept = gated_recurrence(x, g, gate_logits=False, keep=True)
                out = [h, last, kept, *gated_recurrence_grad(x, g, kept, d_h, gate_logits=False)]
                first = first or out
                assert all(torch.equal(p, q) for p, q in zip(out, first)), (t, d, at)


def test_gated_recurrence_decays_above_one_in_some_of_many_histories():
    """More histories than a grid has rows, so that a workgroup walks several: each as if it were alone."""
    from pearl_amd import gated_recurrence, gated_recurrence_grad
    for t, d in ((20, 3), (40, 3), (130, 2)):
        gen = gen_of(t, d, 96)
        b = 65535 + 3000
        x, d_h = rnd(gen, b, t, d), rnd(gen, b, t, d)
        g = (0.9 + 0.05 * torch.rand(b, t, d, generator=gen)).to(DEV)
        grow = torch.zeros(b, dtype=torch.bool)
        grow[torch.randint(0, b, (2000,), generator=gen)] = True
        grow[:1000] = True                       # followed by histories 65535 further on that do not grow,
        grow[1000:2000], grow[66535:67535] = False, True      # and the other way round
        g[grow.to(DEV)] *= 1.3
        g[5, 3:9] = 0.0
        def run(rows):
            h, last, kept = gated_recurrence(x[rows], g[rows], gate_logits=False, keep=True)
            return [h, last, *gated_recurrence_grad(x[rows], g[rows], kept, d_h[rows], gate_logits=False)]
        whole = run(slice(None))
        for rows in (slice(0, 3000), slice(30000, 33000), slice(65000, b)):
            assert all(torch.equal(p[rows], q) for p, q in zip(whole, run(rows))), (t, d, rows)


def test_gated_recurrence_decays_above_one_without_some_gradients():
    from pearl_amd import gated_recurrence, gated_recurrence_grad
    for t in (24, 100, 1500):
        c = growing_case(2, t, 10, torch.float32, torch.float32, 1)
        _, _, kept = gated_recurrence(c["x"], c["g"], c["h0"], gate_logits=False, keep=True)
        zero, none = torch.zeros_like(c["d_h"]), torch.zeros_like(c["d_last"])
        for given, full in (((None, c["d_last"]), (zero, c["d_last"])), ((c["d_h"], None), (c["d_h"], none)),
                            ((None, None), (zero, none))):
            for p, q in zip(gated_recurrence_grad(c["x"], c["g"], kept, *given, gate_logits=False),
                            gated_recurrence_grad(c["x"], c["g"], kept, *full, gate_logits=False)):
                assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("b,t,d", [(2, 30, 9), (2, 120, 9), (3, 250, 65), (1, 2000, 9), (26, 1300, 9), (140, 600, 5)])
def test_gated_recurrence_decays_a_little_above_one(b, t, d, dtype):
    """Products from hardly above one to past 2^60, by channel: some workgroups walk their tiles twice, some chunks
    are joined one after another, others are not."""
    gen = gen_of(b, t, d, 97)
    for reverse in (False, True):
        bits = torch.rand(b, 1, d, generator=gen) * 120.0 / t * torch.randint(0, 2, (b, 1, d), generator=gen)
        up = (torch.rand(b, t, d, generator=gen) < 0.5).double()
        g = torch.exp2(bits * (2 * up - 1))                    # as many steps up as down: the states stay in range
        c = {"x": rnd(gen, b, t, d, dtype=dtype), "g": g.float().to(DEV), "h0": rnd(gen, b, d), "lengths": None,
             "resets": (torch.rand(b, t, generator=gen) < 2.0 / t).to(DEV) if reverse else None,
             "d_h": rnd(gen, b, t, d, dtype=dtype), "d_last": rnd(gen, b, d)}
        check_recurrence(c, False, reverse, dtype, torch.float32, f"reverse {reverse}: ")


@pytest.mark.parametrize("b,t,d", [(2, 30, 8), (2, 120, 8), (1, 900, 8), (30, 700, 8)])
def test_gated_recurrence_half_precision_decays_above_one(b, t, d):
    """Of eight channels: zeros that meet growth; the same, forgotten by a decay of zero; a state of 1e-30 that grows by
    2^100 and shrinks again; ones; minus ones; ordinary ones.  What float16 cannot hold is left out of its gradients."""
    half = t // 2
    grow = 2.0 ** (100.0 / half)
    gen = gen_of(b, t, d, 98)
    x, d_h = torch.randn(b, t, d, generator=gen), torch.randn(b, t, d, generator=gen)
    g = 0.7 + 0.3 * torch.rand(b, t, d, generator=gen)
    h0, d_last = torch.randn(b, d, generator=gen), torch.randn(b, d, generator=gen)
    g[..., 0], x[..., 0], h0[:, 0], d_h[..., 0], d_last[:, 0] = 40.0, 0.0, 0.0, 0.0, 0.0
    g[:, :half, 1], g[:, half, 1], x[:, :half, 1], h0[:, 1], d_h[:, :half, 1] = 60000.0, 0.0, 0.0, 0.0, 0.0
    g[:, :half, 2], g[:, half:, 2], x[..., 2], d_h[..., 2] = grow, 1.0 / grow, 0.0, 0.0
    h0[:, 2] *= 1e-30
    d_last[:, 2] *= 1e-30
    g[..., 3], g[..., 4] = 1.0, -1.0
    for reverse in (False, True):
        turn = (lambda v: v.flip(1)) if reverse else (lambda v: v)
        c = {"x": turn(x).half().to(DEV), "g": turn(g).half().to(DEV), "h0": h0.to(DEV), "d_h": turn(d_h).half().to(DEV),
             "d_last": d_last.to(DEV), "resets": None, "lengths": None}
        from pearl_amd import gated_recurrence, gated_recurrence_grad
        want = O.recurrence(np64(c["x"]), np64(c["g"]), np64(c["h0"]), None, None, False, reverse, np64(c["d_h"]),
                            np64(c["d_last"]))
        # Of the third channel the adjoint, 1e-30 behind the last step, is 1e-30 2^-100 in front of the shrinking
        # half: a float32 holds nothing below 2^-149, so whatever walks the steps may be off by half of that there,
        # and the growing half takes it 2^100 further, to 2^-50 (decays rounded to float16: a factor of 2 at most).
        want["d_h0"][1][:, 2] += 2.0 ** -49
        h, last, kept = gated_recurrence(c["x"], c["g"], c["h0"], gate_logits=False, reverse=reverse, keep=True)
        out = gated_recurrence_grad(c["x"], c["g"], kept, c["d_h"], c["d_last"], gate_logits=False, reverse=reverse)
        for name, got in zip(("h", "last", "d_x", "d_g", "d_h0"), (h, last, *out)):
            kind = torch.float32 if name in ("last", "d_h0") else torch.float16
            O.check(got, *want[name], kind, f"reverse {reverse}: {name}")
