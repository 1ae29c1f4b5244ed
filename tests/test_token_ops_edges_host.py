"""CPU: what the token-policy operators refuse at the edges of their interfaces.  No kernel runs here."""
import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as forward_ad


def recurrence_args(N, **kw):
    buf = C.cast((C.c_char * 65536)(), C.c_void_p).value
    a = N.RecurrenceArgs()
    a.dtype = a.gate_dtype = N.PA_BF16
    a.B, a.T, a.D = 2, 1, 64
    a.x_b = a.gate_b = 64
    a.x, a.gate, a.h0, a.resets, a.lengths, a.h, a.last, a.scratch = (buf + 4096 * k for k in range(8))
    a.resets_b = 1
    a.device = 1000         # what passes the checks ends here
    for k, v in kw.items():
        setattr(a, k, a.last + v[0] if isinstance(v, tuple) else v)
    return a


def test_a_new_state_that_overlaps_what_is_read_is_refused():
    from pearl_amd import _native as N
    lib = N.lib()

    def rc(**kw):
        a = recurrence_args(N, **kw)
        return lib.pa_gated_recurrence(C.byref(a), None)
    passed = N.PA_ERR_HIP
    assert rc() == rc(last=None) == rc(h0=None, resets=None, lengths=None) == passed
    assert rc(h0=(0,)) == passed                                              # a single step in place
    assert rc(h0=(512,)) == rc(h0=(-512,)) == passed                          # side by side
    assert rc(x=(0,), dtype=N.PA_F32, gate_dtype=N.PA_F32) == passed          # read channel by channel as it is written
    assert rc(x=(0,), dtype=N.PA_F32, gate_dtype=N.PA_F32, B=1, x_b=7) == passed
    for bad in (dict(h0=(4,)), dict(h0=(-508,)), dict(h0=(0,), T=2), dict(x=(0,)), dict(x=(-128,)), dict(gate=(0,)),
                dict(x=(0,), dtype=N.PA_F32, gate_dtype=N.PA_F32, x_b=65), dict(resets=(511,)), dict(lengths=(508,)),
                dict(x=(0,), dtype=N.PA_F32, gate_dtype=N.PA_F32, T=2), dict(gate=(-510,), T=3, gate_t=64)):
        assert rc(**bad) == N.PA_ERR_INVALID, bad
        assert "overlaps" in N.last_error()


def test_embedding_gradients_that_would_hold_the_card_are_refused():
    from pearl_amd import _native as N
    lib = N.lib()
    buf = C.cast((C.c_char * 4096)(), C.c_void_p).value

    def rc(n, vocab):
        return lib.pa_embed_tokens_grad(buf, N.PA_F32, 4, buf, N.PA_I64, n, 1.0, vocab, 4, None, buf, 0, None)
    for n, vocab in ((2 ** 26, 2 ** 20), (2 ** 20, 2 ** 26), (2 ** 23, 2 ** 23), (0, 2 ** 26), (1, 1)):
        assert rc(n, vocab) == N.PA_ERR_INVALID          # no place for the result: past the limits
    for n, vocab in ((2 ** 26, 2 ** 20 + 1), (2 ** 20 + 1, 2 ** 26), (2 ** 26, 2 ** 26)):
        assert rc(n, vocab) == N.PA_ERR_UNSUPPORTED and "2^46" in N.last_error()


def test_tangents_are_refused():
    import pearl_amd as P
    from pearl_amd._native import NativeError
    w, tok = torch.randn(5, 4), torch.tensor([0, 1])
    x, row = torch.randn(2, 6, 4), torch.randn(2, 4)
    act, lp = torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    o = P.ActionLogProbs(lp, lp, None, None, torch.zeros(2, 3))
    # every floating-point argument of every entry; plain tensors get as far as "no CPU fallback"
    calls = [(lambda t: P.embed_tokens(t, tok), w), (lambda t: P.embed_tokens_grad(t, tok, 5), row),
             (lambda t: P.gated_recurrence(t, x), x), (lambda t: P.gated_recurrence(x, t), x),
             (lambda t: P.gated_recurrence(x, x, t), row), (lambda t: P.gated_recurrence(t, x, keep=True), x),
             (lambda t: P.gated_recurrence_grad(t, x, w), x), (lambda t: P.gated_recurrence_grad(x, t, w), x),
             (lambda t: P.gated_recurrence_grad(x, x, w, t), x), (lambda t: P.gated_recurrence_grad(x, x, w, x, t), row),
             (lambda t: P.gated_recurrence_step(t, row), row), (lambda t: P.gated_recurrence_step(row, t), row),
             (lambda t: P.gated_recurrence_step(row, row, t), row), (lambda t: P.action_log_probs(t, act), row),
             (lambda t: P.action_log_probs_grad(o, t, act), row), (lambda t: P.action_log_probs_grad(o, row, act, t), lp),
             (lambda t: P.action_log_probs_grad(o, row, act, lp, t), lp)]
    for call, t in calls:
        with pytest.raises(NativeError):
            call(t)
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
            with pytest.raises(NativeError):
                call(t)


def test_temperatures_whose_distances_pass_a_float_are_refused():
    """Above 2^121 the largest distance a float holds, divided by the temperature, no longer underflows in the
    exponential: places that are not available would be counted."""
    from pearl_amd import _native as N, action_log_probs
    lib = N.lib()
    buf = C.cast((C.c_char * 4096)(), C.c_void_p).value

    def rc(entry, temperature):
        a = N.LogProbsArgs()
        a.dtype, a.action_dtype, a.A, a.rows, a.ld, a.temperature, a.device = N.PA_F32, N.PA_I64, 5, 2, 5, temperature, 1000
        a.logits = a.actions = a.log_prob = a.entropy = a.stats = a.d_logits = buf
        return entry(C.byref(a), None)
    for entry in (lib.pa_action_log_probs, lib.pa_action_log_probs_grad):
        assert rc(entry, 2.0 ** 121) == rc(entry, 2.0 ** -126) == N.PA_ERR_HIP      # past the checks
        for far in (2.0 ** 121 * (1 + 2.0 ** -23), 1e37, 1e38, 3.4e38):
            assert rc(entry, far) == N.PA_ERR_INVALID, far
    for far in (2.0 ** 122, 1e38, 1e39, float("inf")):
        with pytest.raises(ValueError):
            action_log_probs(torch.randn(2, 5), torch.zeros(2, dtype=torch.int64), temperature=far)
    assert 3.4028235e38 * 1.4427 / 2.0 ** 121 > 150 > 3.4028235e38 * 1.4427 / 1e38


def test_the_cut_shapes_of_the_gpu_tests_reach_every_way_of_walking_pieces():
    from pearl_amd import _native as N
    from token_cuts import AT_ONCE, CUT_SHAPES, SLAB, cut
    lib = N.lib()
    up = lambda n: -(-n // 256) * 256  # noqa: E731
    reached = set()
    for b, t, d in CUT_SHAPES:
        sizes = []
        for direction in ("forward", "backward"):
            tiles, per_piece, pieces = cut(b, t, d, direction)
            assert pieces > 1
            reached |= {(direction, "several tiles")} if per_piece > 1 else set()
            reached |= {(direction, "several rounds")} if pieces - 1 > AT_ONCE[direction] else set()
            reached |= {(direction, "both")} if per_piece > 1 and pieces - 1 > AT_ONCE[direction] else set()
            # a factor, its exponent and a state per channel, and a byte per slab
            sizes.append(3 * up(b * pieces * d * 4) + up(b * pieces * -(-d // SLAB)))
        assert lib.pa_gated_recurrence_carries(b, t, d) == b * cut(b, t, d, "backward")[0] * d
        assert lib.pa_gated_recurrence_scratch(b, t, d) == max(sizes), (b, t, d)
    assert reached == {(direction, what) for direction in ("forward", "backward")
                       for what in ("several tiles", "several rounds", "both")}


def test_rows_longer_than_the_c_entries_count_are_refused():
    """Their lengths have 32 bits there: 2^32 + 4 columns would have been taken for 4."""
    import pearl_amd as P
    from pearl_amd import _native as N
    tok, act = torch.tensor([0, 0]), torch.zeros(2, dtype=torch.int64)
    for dim in (2 ** 30 + 1, 2 ** 31 + 4, 2 ** 32 + 4):
        with pytest.raises(NotImplementedError):
            P.embed_tokens(torch.zeros(1, 1).expand(1, dim), tok)
    for dim in (2 ** 25 + 1, 2 ** 32 + 4):
        with pytest.raises(NotImplementedError):
            P.embed_tokens_grad(torch.zeros(1, 1).expand(2, dim), tok, 3)
    for width in (2 ** 31, 2 ** 32 + 4):
        with pytest.raises(NotImplementedError):
            P.action_log_probs(torch.zeros(1, 1).expand(2, width), act)
    x = torch.zeros(1, 1, 1).expand(1, 2, 2 ** 32 + 4)
    with pytest.raises(NotImplementedError):
        P.gated_recurrence(x, x)
    with pytest.raises(NotImplementedError):
        P.gated_recurrence_grad(x, x, torch.zeros(1))
    with pytest.raises(NotImplementedError):
        P.gated_recurrence_step(x[:, 0], x[:, 0])
    lib = N.lib()
    buf = C.cast((C.c_char * 4096)(), C.c_void_p).value
    for dim in (2 ** 30 + 1, 2 ** 31 - 1):
        assert lib.pa_embed_tokens(buf, N.PA_F32, 2 ** 32, 8, dim, buf, N.PA_I64, 2, 1.0, buf, 1000, None) == N.PA_ERR_UNSUPPORTED
    for dim in (2 ** 25 + 1, 2 ** 31 - 1):
        assert lib.pa_embed_tokens_grad(buf, N.PA_F32, 2 ** 32, buf, N.PA_I64, 2, 1.0, 8, dim, buf, buf, 1000,
                                        None) == N.PA_ERR_UNSUPPORTED
