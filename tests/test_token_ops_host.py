"""CPU: the token-policy operators' argument checks, their C structs, and the 64-bit definitions that the
GPU tests compare with (gradients against differences).  No kernel runs here."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

import token_oracle as O
from conftest import REPO


def test_ctypes_structs_match_the_header(tmp_path):
    from pearl_amd import _native as N
    pairs = {"pa_recurrence_args": N.RecurrenceArgs, "pa_log_probs_args": N.LogProbsArgs}
    src = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{os.path.join(REPO, "include", "pearl_amd.h")}"',
           'int main(void) {']
    for name, s in pairs.items():
        src.append(f'  printf("%zu", sizeof({name}));')
        src += [f'  printf(" %zu", offsetof({name}, {f[0]}));' for f in s._fields_]
        src.append('  printf("\\n");')
    src += ['  return 0;', '}']
    (tmp_path / "probe.c").write_text("\n".join(src))
    subprocess.run(["gcc", "-std=c99", "-o", str(tmp_path / "probe"), str(tmp_path / "probe.c")], check=True)
    lines = subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.splitlines()
    assert N.RECURRENCE_ARGS.size == C.sizeof(N.RecurrenceArgs) and N.LOG_PROBS_ARGS.size == C.sizeof(N.LogProbsArgs)
    for s, line in zip(pairs.values(), lines):
        assert [int(v) for v in line.split()] == [C.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]


def test_c_entries_refuse_bad_arguments():
    from pearl_amd import _native as N
    lib = N.lib()
    buf = C.cast((C.c_char * 4096)(), C.c_void_p).value
    embed = lambda dtype=N.PA_F32, ldw=4, vocab=8, dim=4, tdt=N.PA_I64, n=2, w=buf, t=buf, o=buf: lib.pa_embed_tokens(  # noqa: E731
        w, dtype, ldw, vocab, dim, t, tdt, n, 1.0, o, 0, None)
    assert embed(n=0) == N.PA_OK
    assert embed(dtype=N.PA_F64) == embed(tdt=N.PA_U8) == N.PA_ERR_UNSUPPORTED
    for bad in (dict(dim=0), dict(vocab=0), dict(vocab=2 ** 33), dict(n=-1), dict(ldw=3), dict(w=None), dict(t=None),
                dict(o=None)):
        assert embed(**bad) == N.PA_ERR_INVALID, bad
    grad = lambda dtype=N.PA_BF16, n=2, vocab=8, dim=4, tdt=N.PA_I32, d=buf, t=buf, w=buf, s=buf, ldd=4: lib.pa_embed_tokens_grad(  # noqa: E731
        d, dtype, ldd, t, tdt, n, 1.0, vocab, dim, w, s, 0, None)
    assert grad(n=2 ** 26 + 1) == grad(vocab=2 ** 26 + 1) == N.PA_ERR_UNSUPPORTED
    assert grad(dtype=N.PA_I64) == grad(tdt=N.PA_F32) == N.PA_ERR_UNSUPPORTED
    for bad in (dict(dim=0), dict(vocab=0), dict(n=-1), dict(d=None), dict(t=None), dict(w=None), dict(s=None), dict(ldd=-1)):
        assert grad(**bad) == N.PA_ERR_INVALID, bad

    def rec(grad=False, **kw):
        a = N.RecurrenceArgs()
        a.dtype = a.gate_dtype = N.PA_BF16
        a.B, a.T, a.D = 2, 3, 4
        a.x = a.gate = a.h = a.d_x = a.d_gate = a.carries = a.scratch = buf
        for k, v in kw.items():
            setattr(a, k, v)
        return (lib.pa_gated_recurrence_grad if grad else lib.pa_gated_recurrence)(C.byref(a), None)
    assert rec(B=0) == rec(True, B=0) == N.PA_OK
    assert rec(dtype=N.PA_I64) == rec(gate_dtype=N.PA_F16) == rec(dtype=N.PA_F32) == N.PA_ERR_UNSUPPORTED
    for far in (dict(x_t=2 ** 22), dict(gate_t=2 ** 22), dict(resets_t=2 ** 23), dict(d_h_t=2 ** 22), dict(x_t=-1), dict(D=2 ** 21)):
        assert rec(**far) == N.PA_ERR_UNSUPPORTED, far
    for bad in (dict(T=0), dict(D=0), dict(B=-1), dict(x=None), dict(gate=None), dict(h=None), dict(B=2 ** 40),
                dict(B=1, T=4000, scratch=None)):
        assert rec(**bad) == N.PA_ERR_INVALID, bad
    for bad in (dict(carries=None), dict(d_x=None), dict(d_gate=None)):
        assert rec(True, **bad) == N.PA_ERR_INVALID, bad
    assert lib.pa_gated_recurrence(None, None) == lib.pa_action_log_probs(None, None) == N.PA_ERR_INVALID

    def lp(grad=False, **kw):
        a = N.LogProbsArgs()
        a.dtype, a.action_dtype, a.A, a.rows, a.ld, a.temperature = N.PA_F16, N.PA_I64, 5, 2, 5, 1.0
        a.logits = a.actions = a.log_prob = a.entropy = a.stats = a.d_logits = buf
        for k, v in kw.items():
            setattr(a, k, v)
        return (lib.pa_action_log_probs_grad if grad else lib.pa_action_log_probs)(C.byref(a), None)
    assert lp(rows=0) == lp(True, rows=0) == N.PA_OK
    assert lp(dtype=N.PA_U8) == lp(action_dtype=N.PA_F32) == lp(top=65) == lp(top=-1) == N.PA_ERR_UNSUPPORTED
    for bad in (dict(A=0), dict(rows=-1), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(temperature=float("inf")), dict(temperature=1e-40), dict(logits=None), dict(actions=None),
                dict(log_prob=None), dict(entropy=None), dict(top=3), dict(A=100000, scratch=None), dict(ld=-5)):
        assert lp(**bad) == N.PA_ERR_INVALID, bad
    for bad in (dict(stats=None), dict(d_logits=None)):
        assert lp(True, **bad) == N.PA_ERR_INVALID, bad


def test_python_entries_refuse_bad_arguments_and_cpu_tensors():
    import pearl_amd as P
    from pearl_amd._native import NativeError
    w, tok = torch.randn(5, 4), torch.tensor([0, 1])
    with pytest.raises(ValueError):
        P.embed_tokens(w[0], tok)
    with pytest.raises(TypeError):
        P.embed_tokens(w.double(), tok)
    with pytest.raises(TypeError):
        P.embed_tokens(w, tok.float())
    with pytest.raises(NativeError):
        P.embed_tokens(w, tok)
    with pytest.raises(ValueError):
        P.embed_tokens_grad(w, tok, 5)
    with pytest.raises(NativeError):
        P.embed_tokens_grad(w[:2], tok, 5)
    x, g = torch.randn(2, 6, 4), torch.randn(2, 6, 4)
    bad = [(ValueError, (x[0], g[0])), (ValueError, (x, g[:, :5])), (TypeError, (x.double(), g.double())),
           (TypeError, (x, g.half())), (TypeError, (x.half(), g.bfloat16())),
           (ValueError, (x, g, torch.zeros(2, 5))), (ValueError, (x, g, torch.zeros(2, 4).half())),
           (ValueError, (x, g, None, torch.zeros(2, 6))), (ValueError, (x, g, None, torch.zeros(2, 5).bool())),
           (ValueError, (x, g, None, None, torch.zeros(2))), (ValueError, (x, g, None, None, torch.zeros(3).int())),
           (NativeError, (x, g))]
    for kind, args in bad:
        with pytest.raises(kind):
            P.gated_recurrence(*args)
    for kind, kw in [(ValueError, dict(d_h=g[:, :5])), (ValueError, dict(d_h=g.half())), (ValueError, dict(d_last=g[:, 0].half())),
                     (NativeError, dict(d_h=g))]:
        with pytest.raises(kind):
            P.gated_recurrence_grad(x, g, torch.zeros(1), **kw)
    with pytest.raises(RuntimeError):
        P.gated_recurrence_step(x[:, 0].clone().requires_grad_(), g[:, 0])
    with pytest.raises(ValueError):
        P.gated_recurrence_step(x, g)
    with pytest.raises(ValueError):
        P.gated_recurrence_step(x[:, 0], g[:, 0], resets=torch.zeros(2, 1).bool())
    with pytest.raises(NativeError):
        P.gated_recurrence_step(x[:, 0], g[:, 0])
    lg, act = torch.randn(3, 7), torch.zeros(3, dtype=torch.int64)
    for kind, args, kw in [(ValueError, (lg, act[:2]), {}), (TypeError, (lg.double(), act), {}), (TypeError, (lg, act.float()), {}),
                           (ValueError, (lg, act, torch.zeros(3, 6).bool()), {}), (ValueError, (lg, act, torch.zeros(3, 7)), {}),
                           (ValueError, (lg, act), dict(temperature=0.0)), (ValueError, (lg, act), dict(temperature=float("nan"))),
                           (NotImplementedError, (lg, act), dict(top=65)), (NativeError, (lg, act), {})]:
        with pytest.raises(kind):
            P.action_log_probs(*args, **kw)


def _differences(f, arrays, k, step=1e-6):
    out = np.zeros_like(arrays[k])
    for i in np.ndindex(out.shape):
        up, down = [a.copy() for a in arrays], [a.copy() for a in arrays]
        up[k][i] += step
        down[k][i] -= step
        out[i] = (f(*up) - f(*down)) / (2 * step)
    return out


@pytest.mark.parametrize("logits", [True, False])
@pytest.mark.parametrize("reverse", [True, False])
def test_recurrence_definition_against_differences(logits, reverse):
    rng = np.random.default_rng(0)
    x, g, d_h = (rng.normal(size=(2, 7, 3)) for _ in range(3))
    h0, d_last = rng.normal(size=(2, 3)), rng.normal(size=(2, 3))
    resets, lengths = rng.random((2, 7)) < 0.25, [7, 4]

    def loss(x, g, h0):
        o = O.recurrence(x, g, h0, resets, lengths, logits, reverse)
        return (o["h"][0] * d_h).sum() + (o["last"][0] * d_last).sum()
    want = O.recurrence(x, g, h0, resets, lengths, logits, reverse, d_h, d_last)
    for k, name in enumerate(("d_x", "d_g", "d_h0")):
        np.testing.assert_allclose(want[name][0], _differences(loss, [x, g, h0], k), rtol=1e-6, atol=1e-8)


def test_log_prob_definition_against_differences():
    rng = np.random.default_rng(1)
    logits, mask, actions = rng.normal(size=(4, 6)), rng.random((4, 6)) < 0.3, np.array([0, 5, -1, 2])
    mask[0, 0] = mask[3, 2] = False
    mask[1, 5] = True
    g_lp, g_h = rng.normal(size=4), rng.normal(size=4)

    def loss(logits):
        o = O.log_probs(logits, actions, mask, 0.7, 0)
        lp = np.where(np.isinf(o["log_prob"][0]), 0.0, o["log_prob"][0])
        return (lp * g_lp).sum() + (o["entropy"][0] * g_h).sum()
    want = O.log_probs(logits, actions, mask, 0.7, 0, g_lp, g_h)["d_logits"][0]
    np.testing.assert_allclose(want, _differences(loss, [logits], 0), rtol=1e-6, atol=1e-8)


def test_embedding_gradient_definition_against_differences():
    rng = np.random.default_rng(2)
    w, d, tok = rng.normal(size=(4, 3)), rng.normal(size=(6, 3)), np.array([0, 3, 3, -1, 9, 0])

    def loss(w):
        return (np.nan_to_num(O.embed(w, tok, 1.5)[0]) * d).sum()
    np.testing.assert_allclose(O.embed_grad(d, tok, 4, 1.5)[0], _differences(loss, [w], 0), rtol=1e-6, atol=1e-8)


def test_recurrent_actor_network_constructor():
    from pearl_amd import RecurrentActorNetwork
    net = RecurrentActorNetwork(12, [8], 5)
    assert sorted(net.state_dict()) == ["_embedding", "_head.bias", "_head.weight", "_inputs.bias", "_inputs.weight"]
    assert net.initial_state(3).shape == (3, 8)
    for hidden in (None, [], [4, 4]):
        with pytest.raises(ValueError):
            RecurrentActorNetwork(12, hidden, 5)
    with pytest.raises(NotImplementedError):
        net.linear_layers()
