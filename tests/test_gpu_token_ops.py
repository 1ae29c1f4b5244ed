"""The token-policy operators on the GPU against their 64-bit definitions (tests/token_oracle.py)."""
import math

import numpy as np
import pytest
import torch

import token_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]
DEV = "cuda:0"


def np64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def rnd(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(DEV)


def gen_of(*key):
    return torch.Generator().manual_seed(abs(hash(key)) % (2 ** 31) if not all(isinstance(k, int) for k in key)
                                         else sum(k * 7919 ** i for i, k in enumerate(key)) % (2 ** 31))


# ---------------------------------------------------------------------------- embedding
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (5, 7, 3), (64, 16, 128), (33, 1003, 333), (129, 50, 2049),
                                         (1000, 40, 8)])
def test_embed_tokens(dtype, n, vocab, dim):
    from pearl_amd import embed_tokens
    gen = gen_of(n, vocab, dim)
    w = rnd(gen, vocab, dim, dtype=dtype)
    tok = torch.randint(0, vocab, (n,), generator=gen)
    tok[n // 2] = -1 if n > 1 else 0
    for index in (torch.int64, torch.int32):
        for scale in (1.0, math.sqrt(dim)):
            out = embed_tokens(w, tok.to(DEV, index), scale=scale)
            value, bound = O.embed(np64(w), tok.numpy(), scale)
            assert out.dtype == dtype
            O.check(out, value, bound, dtype, "embed")
    assert torch.equal(embed_tokens(w, tok.clamp(min=0).to(DEV)), w[tok.clamp(min=0).to(DEV)])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_embed_tokens_outside_the_table_and_strided(dtype):
    from pearl_amd import embed_tokens
    gen = gen_of(3)
    wide = rnd(gen, 20, 101, dtype=dtype)
    w = wide[:, 3:72]                             # rows 101 elements apart, from an odd element on
    tok = torch.tensor([[0, 19, 20], [-1, -2, 2 ** 40]])
    out = embed_tokens(w, tok.to(DEV), scale=0.5)
    assert out.shape == (2, 3, 69)
    value, bound = O.embed(np64(w), tok.numpy(), 0.5)
    O.check(out, value, bound, dtype, "embed")
    assert torch.isnan(out[0, 2]).all() and (out[1, 0] == 0).all()
    every_other = wide[:, ::2]                    # not contiguous in a row
    O.check(embed_tokens(every_other, tok.to(DEV)), *O.embed(np64(every_other), tok.numpy(), 1.0), dtype, "columns")
    one_row = w[:1].expand(20, 69)                # the same row for every token
    O.check(embed_tokens(one_row, tok.to(DEV)), *O.embed(np64(one_row), tok.numpy(), 1.0), dtype, "expanded")
    assert embed_tokens(w, torch.empty(0, 4, dtype=torch.int64, device=DEV)).shape == (0, 4, 69)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,vocab,dim,kind", [(1, 1, 1, "any"), (1, 300, 5, "any"), (7, 4, 3, "any"),
                                              (64, 1, 17, "same"), (65, 9, 130, "any"), (700, 30, 333, "skew"),
                                              (1500, 5000, 40, "any"), (2100, 3, 2050, "same"), (4099, 700, 24, "skew"),
                                              (9000, 17, 12, "none"),
                                              (20000, 70000, 6, "skew"), (40000, 5, 3, "same")])
def test_embed_grad(dtype, n, vocab, dim, kind):
    from pearl_amd import embed_tokens_grad
    gen = gen_of(n, vocab, dim, 1)
    tok = torch.randint(0, vocab, (n,), generator=gen)
    if kind == "same":
        tok[:] = vocab - 1
        if n > 100:
            tok[n // 3] = 0
    if kind == "skew":
        tok = (torch.rand(n, generator=gen) ** 6 * vocab).long()
    if kind == "none":
        tok[torch.rand(n, generator=gen) < 0.3] = -1
        tok[::97] = vocab + 5
        tok[::89] = -7
    d = rnd(gen, n, dim, dtype=dtype)
    d[((tok < 0) | (tok >= vocab)).to(DEV)] = float("nan")        # rows without a token take no part
    value, bound = O.embed_grad(np64(d), tok.numpy(), vocab, 1.7)
    for index in (torch.int64, torch.int32):
        got = embed_tokens_grad(d, tok.to(DEV, index), vocab, scale=1.7)
        assert got.dtype == dtype
        O.check(got, value, bound, dtype, "embed grad")
    again = embed_tokens_grad(d, tok.to(DEV), vocab, scale=1.7)
    assert torch.equal(got, again)


def test_embed_grad_without_tokens_clears_the_table():
    from pearl_amd import embed_tokens_grad
    for dtype in DTYPES:
        d = embed_tokens_grad(torch.empty(0, 5, dtype=dtype, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV), 7)
        assert d.shape == (7, 5) and d.dtype == dtype and (d == 0).all()
        none = torch.full((3,), -1, device=DEV)
        assert (embed_tokens_grad(torch.full((3, 5), float("nan"), dtype=dtype, device=DEV), none, 7) == 0).all()


def test_embed_grad_strided_and_broadcast_gradients():
    from pearl_amd import embed_tokens, embed_tokens_grad
    gen = gen_of(11)
    tok = torch.randint(0, 13, (6, 50), generator=gen)
    wide = rnd(gen, 6, 50, 77, dtype=torch.bfloat16)
    d = wide[..., 5:30]
    O.check(embed_tokens_grad(d, tok.to(DEV), 13), *O.embed_grad(np64(d), tok.numpy(), 13, 1.0), torch.bfloat16, "slice")
    flat = wide.view(300, 77)[:, 5:30]
    O.check(embed_tokens_grad(flat, tok.view(-1).to(DEV), 13), *O.embed_grad(np64(d), tok.numpy(), 13, 1.0),
            torch.bfloat16, "row stride")
    one = rnd(gen, 1, 25).expand(300, 25)
    O.check(embed_tokens_grad(one, tok.view(-1).to(DEV), 13), *O.embed_grad(np64(one), tok.view(-1).numpy(), 13, 1.0),
            torch.float32, "expanded")
    w = rnd(gen, 13, 25).requires_grad_()
    (embed_tokens(w, tok.to(DEV), scale=3.0) * d.float()).sum().backward()
    O.check(w.grad, *O.embed_grad(np64(d), tok.numpy(), 13, 3.0), torch.float32, "autograd")
    w.grad = None
    embed_tokens(w, tok.to(DEV)).sum().backward()           # an expanded gradient
    counts = torch.bincount(tok.view(-1), minlength=13).float()
    assert torch.equal(w.grad.cpu(), counts[:, None].expand(13, 25))


# ---------------------------------------------------------------------------- recurrence
def recurrence_case(b, t, d, dtype, gate_dtype, logits, key, h0=True, resets=True, lengths=False):
    gen = gen_of(b, t, d, key)
    x = rnd(gen, b, t, d, dtype=dtype)
    g = rnd(gen, b, t, d) * 2 + 1 if logits else (0.7 + 0.3 * torch.rand(b, t, d, generator=gen)).to(DEV)
    case = {"x": x, "g": g.to(gate_dtype), "h0": rnd(gen, b, d) if h0 else None,
            "resets": (torch.rand(b, t, generator=gen) < 0.05).to(DEV) if resets else None,
            "lengths": torch.randint(0, t + 1, (b,), generator=gen).to(DEV) if lengths else None,
            "d_h": rnd(gen, b, t, d, dtype=dtype), "d_last": rnd(gen, b, d)}
    if lengths and b > 1:
        case["lengths"][0], case["lengths"][1] = 0, t
    return case


def check_recurrence(c, logits, reverse, dtype, gate_dtype, what=""):
    from pearl_amd import gated_recurrence, gated_recurrence_grad
    want = O.recurrence(np64(c["x"]), np64(c["g"]), np64(c["h0"]), None if c["resets"] is None else c["resets"].cpu(),
                        None if c["lengths"] is None else c["lengths"].cpu(), logits, reverse, np64(c["d_h"]),
                        np64(c["d_last"]))
    how = dict(resets=c["resets"], lengths=c["lengths"], gate_logits=logits, reverse=reverse)
    h, last = gated_recurrence(c["x"], c["g"], c["h0"], **how)
    O.check(h, *want["h"], dtype, what + "h")
    O.check(last, *want["last"], torch.float32, what + "last")
    h2, last2, kept = gated_recurrence(c["x"], c["g"], c["h0"], keep=True, **how)
    dx, dg, d0 = gated_recurrence_grad(c["x"], c["g"], kept, c["d_h"], c["d_last"], **how)
    O.check(h2, *want["h"], dtype, what + "kept h")
    O.check(last2, *want["last"], torch.float32, what + "kept last")
    O.check(dx, *want["d_x"], dtype, what + "d_x")
    O.check(dg, *want["d_g"], gate_dtype, what + "d_gate")
    O.check(d0, *want["d_h0"], torch.float32, what + "d_initial")
    assert dx.dtype == dtype and dg.dtype == gate_dtype and h.dtype == dtype


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("logits", [True, False], ids=["logit", "decay"])
@pytest.mark.parametrize("b,t,d", [(1, 1, 1), (3, 1, 70), (2, 2, 5), (2, 31, 64), (2, 32, 65), (3, 33, 9), (1, 257, 40),
                                   (2, 300, 129), (1, 1500, 17), (2, 128, 40), (1, 129, 33), (1, 256, 2), (2, 1030, 66)])
def test_gated_recurrence(dtype, logits, b, t, d):
    for k, (reverse, resets, lengths) in enumerate([(False, False, False), (True, True, False), (False, True, True),
                                                    (True, False, True)]):
        c = recurrence_case(b, t, d, dtype, dtype, logits, k, h0=k != 1, resets=resets, lengths=lengths)
        check_recurrence(c, logits, reverse, dtype, dtype, f"reverse {reverse} resets {resets} lengths {lengths}: ")


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
def test_gated_recurrence_float_gates(dtype):
    for logits in (True, False):
        c = recurrence_case(2, 290, 75, dtype, torch.float32, logits, 5, lengths=True)
        check_recurrence(c, logits, False, dtype, torch.float32)
        check_recurrence(c, logits, True, dtype, torch.float32)


def test_gated_recurrence_one_workgroup_per_history_walks_all_tiles():
    # 200 histories: no cut of the steps; three tiles each
    c = recurrence_case(200, 600, 8, torch.float32, torch.float32, True, 6, lengths=True)
    check_recurrence(c, True, False, torch.float32, torch.float32)


def test_gated_recurrence_strided_inputs():
    gen = gen_of(21)
    both = rnd(gen, 2, 70, 2 * 37 + 1, dtype=torch.bfloat16)
    c = recurrence_case(2, 70, 37, torch.bfloat16, torch.bfloat16, True, 9)
    c["x"], c["g"] = both[..., 1:38], both[..., 38:]          # the two halves of one projection, odd offsets
    check_recurrence(c, True, False, torch.bfloat16, torch.bfloat16, "halves: ")
    c["x"] = rnd(gen, 70, 2, 37, dtype=torch.bfloat16).transpose(0, 1)     # time-major
    c["d_h"] = rnd(gen, 1, 1, 37, dtype=torch.bfloat16).expand(2, 70, 37)
    c["resets"] = (torch.rand(70, 2, generator=gen) < 0.1).to(DEV).t()
    check_recurrence(c, True, True, torch.bfloat16, torch.bfloat16, "time-major: ")
    c["g"] = rnd(gen, 37, dtype=torch.bfloat16).expand(2, 70, 37)          # one gate for all steps
    check_recurrence(c, True, False, torch.bfloat16, torch.bfloat16, "one gate: ")
    c["x"] = rnd(gen, 2, 37, 70, dtype=torch.bfloat16).transpose(1, 2)     # channels not adjacent
    check_recurrence(c, True, False, torch.bfloat16, torch.bfloat16, "channels: ")
    far = torch.zeros(70, 2 ** 22 + 5, dtype=torch.bfloat16, device=DEV)[:, :37]     # steps 8 MB apart
    far.copy_(rnd(gen, 70, 37, dtype=torch.bfloat16))
    c["x"] = far.unsqueeze(0).expand(2, 70, 37)
    check_recurrence(c, True, True, torch.bfloat16, torch.bfloat16, "far: ")


def test_gated_recurrence_resets_forget_and_padding_hides_anything():
    from pearl_amd import gated_recurrence, gated_recurrence_grad
    for t in (20, 300, 1100):
        for logits in (True, False):
            c = recurrence_case(2, t, 33, torch.float32, torch.float32, logits, 31, resets=False)
            r = torch.zeros(2, t, dtype=torch.bool, device=DEV)
            r[:, t // 2] = True
            ends = torch.tensor([t - 3, t - 1], device=DEV)
            clean = dict(x=c["x"].clone(), g=c["g"].clone())
            dirty = dict(x=c["x"].clone(), g=c["g"].clone())
            dirty["x"][:, t // 2 - 2] = float("inf")          # in the episode before the reset
            dirty["x"][:, t // 2 - 1, ::2] = float("nan")
            d_dirty = c["d_h"].clone()
            for i, e in enumerate(ends.tolist()):
                dirty["x"][i, e:], dirty["g"][i, e:], d_dirty[i, e:] = float("nan"), float("inf"), float("nan")
            how = dict(resets=r, lengths=ends, gate_logits=logits)
            h, last, kept = gated_recurrence(clean["x"], clean["g"], c["h0"], keep=True, **how)
            h2, last2, kept2 = gated_recurrence(dirty["x"], dirty["g"], c["h0"], keep=True, **how)
            assert torch.equal(h[:, t // 2:], h2[:, t // 2:]) and torch.equal(last, last2)
            assert torch.isfinite(h2[:, t // 2:]).all() and not torch.isfinite(h2[:, t // 2 - 1]).any()
            g1 = gated_recurrence_grad(clean["x"], clean["g"], kept, c["d_h"], c["d_last"], **how)
            g2 = gated_recurrence_grad(dirty["x"], dirty["g"], kept2, d_dirty, c["d_last"], **how)
            for a, b in zip(g1[:2], g2[:2]):
                assert torch.equal(a[:, t // 2 + 1:], b[:, t // 2 + 1:]) and torch.isfinite(b[:, t // 2 + 1:]).all()
            assert torch.equal(g1[1][:, t // 2], g2[1][:, t // 2])
            for i, e in enumerate(ends.tolist()):
                assert (h2[i, e:] == 0).all() and (g2[0][i, e:] == 0).all() and (g2[1][i, e:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gated_recurrence_saturated_gates(dtype):
    """Gates far out, infinite among them: the state is kept or replaced, nothing turns into NaN."""
    from pearl_amd import gated_recurrence, gated_recurrence_grad
    inf = float("inf")
    x = rnd(gen_of(71), 1, 8, 20, dtype=dtype)
    h0 = rnd(gen_of(72), 1, 20)
    g = torch.tensor([200.0, inf, -200.0, 1e4, inf, -inf, 87.5, -87.5], device=DEV).to(dtype).view(1, 8, 1).expand(1, 8, 20)
    h, last, kept = gated_recurrence(x, g, h0, keep=True)
    want = torch.stack([h0, h0, x[:, 2].float(), x[:, 2].float(), x[:, 2].float(), x[:, 5].float(), x[:, 5].float(), x[:, 7].float()], 1)
    assert float((last - want[:, -1]).abs().max()) < 1e-30
    assert torch.equal(h.float(), want.to(dtype).float())
    d = rnd(gen_of(73), 1, 8, 20, dtype=dtype)
    dx, dg, d0 = gated_recurrence_grad(x, g, kept, d)
    assert float(dg.float().abs().max()) < 1e-30
    torch.testing.assert_close(d0, (d[:, 0].float() + d[:, 1].float()), rtol=4 * O.U, atol=0)
    # a sum of three in fp32 is off by at most 2 U times the sum of their sizes in either order, so two orders
    # differ by 4 U of it, and by one rounding to the type each
    three = d[:, 2:5].double().cpu()
    far = (dx[:, 2].double().cpu() - three.sum(1)).abs()
    assert (far <= 4 * O.U * three.abs().sum(1) + torch.finfo(dtype).eps * three.sum(1).abs()).all()
    # a NaN gate shows in its own channel from its step on, and nowhere else
    bad = g.clone()
    bad[0, 4, 3] = float("nan")
    h, _ = gated_recurrence(x, bad, h0)
    assert torch.isnan(h[0, 4:, 3]).all() and torch.isfinite(h[0, :4]).all() and torch.isfinite(h[0, :, :3]).all()


def test_gated_recurrence_autograd_matches_explicit_gradients():
    from pearl_amd import gated_recurrence, gated_recurrence_grad
    c = recurrence_case(3, 100, 40, torch.float32, torch.float32, True, 41, lengths=True)
    how = dict(resets=c["resets"], lengths=c["lengths"])
    _, _, kept = gated_recurrence(c["x"], c["g"], c["h0"], keep=True, **how)
    for use_h, use_last in ((True, True), (True, False), (False, True)):
        leaves = [c[k].clone().requires_grad_() for k in ("x", "g", "h0")]
        h, last = gated_recurrence(*leaves, **how)
        loss = (h * c["d_h"]).sum() * use_h + (last * c["d_last"]).sum() if use_last else (h * c["d_h"]).sum()
        if not use_h:
            loss = (last * c["d_last"]).sum()
        loss.backward()
        want = gated_recurrence_grad(c["x"], c["g"], kept, c["d_h"] if use_h else None,
                                     c["d_last"] if use_last else None, **how)
        for leaf, w in zip(leaves, want):
            assert torch.equal(leaf.grad, w)
    # one gate for every step and history: its gradient is the sum over them
    gate = rnd(gen_of(43), 40).requires_grad_()
    h, _ = gated_recurrence(c["x"], gate.expand(3, 100, 40), c["h0"], **how)
    (h * c["d_h"]).sum().backward()
    w = O.recurrence(np64(c["x"]), np64(gate.expand(3, 100, 40)), np64(c["h0"]), c["resets"].cpu(), c["lengths"].cpu(),
                     True, False, np64(c["d_h"]))["d_g"]
    O.check(gate.grad, w[0].sum((0, 1)), w[1].sum((0, 1)) + 300 * O.U * np.abs(w[0]).sum((0, 1)), torch.float32, "shared gate")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gated_recurrence_step_continues_a_history(dtype):
    from pearl_amd import gated_recurrence, gated_recurrence_step
    for logits in (True, False):
        c = recurrence_case(5, 12, 67, dtype, dtype, logits, 51)
        want = O.recurrence(np64(c["x"]), np64(c["g"]), np64(c["h0"]), c["resets"].cpu(), None, logits, False)
        state = c["h0"].clone()
        for t in range(12):
            h, out = gated_recurrence_step(c["x"][:, t], c["g"][:, t], state, resets=c["resets"][:, t],
                                           gate_logits=logits, out_state=state)
            assert out is state
            O.check(h, want["h"][0][:, t], want["h"][1][:, t], dtype, f"step {t}")
        O.check(state, *want["last"], torch.float32, "state")
        h, new = gated_recurrence_step(c["x"][:, 0], c["g"][:, 0], gate_logits=logits)
        h1, last1 = gated_recurrence(c["x"][:, :1], c["g"][:, :1], gate_logits=logits)
        assert torch.equal(h, h1[:, 0]) and torch.equal(new, last1)


def test_gated_recurrence_empty_sizes():
    from pearl_amd import gated_recurrence
    h0 = torch.randn(3, 8, device=DEV)
    h, last = gated_recurrence(torch.empty(3, 0, 8, device=DEV), torch.empty(3, 0, 8, device=DEV), h0)
    assert h.shape == (3, 0, 8) and torch.equal(last, h0) and last.data_ptr() != h0.data_ptr()
    h, last = gated_recurrence(torch.empty(0, 5, 8, device=DEV), torch.empty(0, 5, 8, device=DEV))
    assert h.shape == (0, 5, 8) and last.shape == (0, 8)
    leaf = h0.clone().requires_grad_()
    _, last = gated_recurrence(torch.empty(3, 0, 8, device=DEV), torch.empty(3, 0, 8, device=DEV), leaf)
    (last * 2).sum().backward()
    assert (leaf.grad == 2).all()


# ---------------------------------------------------------------------------- log probabilities
def check_log_probs(logits, actions, mask, temperature, top, dtype, g_lp, g_h, what=""):
    from pearl_amd import action_log_probs, action_log_probs_grad
    width = logits.shape[-1]
    full = None if mask is None else mask.expand(logits.shape).cpu().numpy()
    want = O.log_probs(np64(logits), actions.cpu().numpy(), full, temperature, top, np64(g_lp), np64(g_h))
    for index in (torch.int64, torch.int32):
        o = action_log_probs(logits, actions.to(index), mask, temperature=temperature, top=top)
        O.check(o.log_prob, *want["log_prob"], torch.float32, what + "log_prob")
        O.check(o.entropy, *want["entropy"], torch.float32, what + "entropy")
        if top:
            assert np.array_equal(o.top_actions.cpu().numpy(), want["top"]), what + "alternatives"
            O.check(o.top_log_probs, *want["top_log_prob"], torch.float32, what + "alternatives' log_prob")
        else:
            assert o.top_actions is None and o.top_log_probs is None
    d = action_log_probs_grad(o, logits, actions, g_lp, g_h, mask, temperature)
    assert d.dtype == dtype and d.shape == logits.shape and width
    O.check(d, *want["d_logits"], dtype, what + "d_logits")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 2), (5, 5), (64, 16), (7, 129), (3, 256), (4, 257), (9, 1000), (2, 4097),
                                        (600, 300), (515, 4200), (3, 20011), (1, 70001)])
def test_action_log_probs(dtype, rows, width):
    gen = gen_of(rows, width)
    logits = rnd(gen, rows, width, dtype=dtype, scale=3.0)
    actions = torch.randint(0, width, (rows,), generator=gen).to(DEV)
    g_lp, g_h = rnd(gen, rows), rnd(gen, rows)
    check_log_probs(logits, actions, None, 1.0, 0, dtype, g_lp, g_h, "plain: ")
    check_log_probs(logits, actions, None, 0.7, min(20, width), dtype, g_lp, None, "top: ")
    mask = (torch.rand(rows, width, generator=gen) < 0.4).to(DEV)
    mask[rows // 2] = True                                     # a row with nothing
    actions[0] = -1
    check_log_probs(logits, actions, mask, 1.6, 64 if rows < 100 else 3, dtype, None, g_h, "mask: ")
    check_log_probs(logits, actions, mask[0].clone(), 1.0, 1, dtype, g_lp, g_h, "one mask: ")


@pytest.mark.parametrize("width", [16, 300, 5000, 40000])
def test_action_log_probs_ties_go_to_the_lowest_index(width):
    gen = gen_of(width, 77)
    for rows in (6, 700 if width == 300 else 6):
        logits = torch.randint(-2, 3, (rows, width), generator=gen).to(torch.bfloat16).to(DEV)
        logits[0] = 1.5                                       # all the same
        logits[1] = torch.arange(width, device=DEV).to(torch.bfloat16) / 256    # rising: every value passes the last
        logits[2, ::2] = 0.0
        logits[2, 1::2] = -0.0                                # equal
        actions = torch.zeros(rows, dtype=torch.int64, device=DEV)
        for top in (1, 7, 64):
            check_log_probs(logits, actions, None, 1.0, top, torch.bfloat16, None, None, f"top {top}: ")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("width", [10, 400, 9000])
def test_action_log_probs_odd_values(dtype, width):
    gen = gen_of(width, 78)
    low = torch.finfo(dtype).min
    logits = rnd(gen, 12, width, dtype=dtype, scale=2.0)
    mask = torch.zeros(12, width, dtype=torch.bool, device=DEV)
    actions = torch.full((12,), 2, device=DEV)
    mask[0, 1], logits[0, 1] = True, float("nan")             # hidden places hold anything
    mask[1, 1], logits[1, 1] = True, float("inf")
    logits[2, 3:] = low                                       # masks added as the lowest value
    logits[3, :] = low                                        # ... everywhere: all equally probable
    logits[4, :] = float("-inf")                              # nothing left
    logits[5, 2] = float("-inf")                              # the action taken is unavailable
    mask[6, 2] = True
    logits[7, 4] = float("nan")
    logits[8, 4] = float("inf")
    actions[9], actions[10] = width, -5                       # outside
    logits[11] = 0
    logits[11, 2] = 60.0 if dtype != torch.float32 else 200.0   # all the rest underflows
    g_lp, g_h = rnd(gen, 12), rnd(gen, 12)
    check_log_probs(logits, actions, mask, 1.0, 5, dtype, g_lp, g_h)
    check_log_probs(logits, actions, mask, 2.5, 0, dtype, g_lp, None)


def test_action_log_probs_strided_and_batched():
    from pearl_amd import action_log_probs
    gen = gen_of(5)
    wide = rnd(gen, 6, 9, 413, dtype=torch.float16, scale=2.0)
    logits = wide[..., 3:402]
    actions = torch.randint(0, 399, (6, 9), generator=gen).to(DEV)
    mask = (torch.rand(6, 9, 800, generator=gen) < 0.2).to(DEV)[..., ::2][..., :399]
    o = action_log_probs(logits, actions, mask, top=4)
    w = O.log_probs(np64(logits).reshape(54, 399), actions.view(-1).cpu().numpy(), mask.reshape(54, 399).cpu().numpy(), 1.0, 4)
    O.check(o.log_prob.reshape(-1), *w["log_prob"], torch.float32, "log_prob")
    assert o.top_actions.shape == (6, 9, 4) and np.array_equal(o.top_actions.view(54, 4).cpu().numpy(), w["top"])
    flat = wide.view(54, 413)[:, 3:402]
    check_log_probs(flat, actions.view(-1), mask.reshape(54, 399), 1.0, 4, torch.float16, None, None, "row stride: ")
    shared = rnd(gen, 1, 399).expand(54, 399)
    check_log_probs(shared, actions.view(-1), None, 1.0, 2, torch.float32, rnd(gen, 54), None, "one row: ")
    one = action_log_probs(logits[0, 0], actions[0, 0])
    O.check(one.log_prob, *(v[0] for v in O.log_probs(np64(logits[0, :1]), actions[0, :1].cpu().numpy(), None, 1.0, 0)["log_prob"]),
            torch.float32, "one position")
    empty = action_log_probs(logits[:0], actions[:0], top=3)
    assert empty.log_prob.shape == (0, 9) and empty.top_actions.shape == (0, 9, 3)


def test_action_log_probs_autograd():
    from pearl_amd import action_log_probs, action_log_probs_grad
    gen = gen_of(6)
    for width in (16, 700):
        logits = rnd(gen, 5, 4, width)
        actions = torch.randint(0, width, (5, 4), generator=gen).to(DEV)
        g_lp, g_h = rnd(gen, 5, 4), rnd(gen, 5, 4)
        o = action_log_probs(logits, actions, temperature=0.8)
        for use_lp, use_h in ((True, True), (True, False), (False, True)):
            leaf = logits.clone().requires_grad_()
            out = action_log_probs(leaf, actions, temperature=0.8, top=3)
            assert not out.top_log_probs.requires_grad and out.log_prob.requires_grad
            outs = [v for v, on in ((out.log_prob, use_lp), (out.entropy, use_h)) if on]
            torch.autograd.backward(outs, [v for v, on in ((g_lp, use_lp), (g_h, use_h)) if on])
            want = action_log_probs_grad(o, logits, actions, g_lp if use_lp else None, g_h if use_h else None, None, 0.8)
            assert torch.equal(leaf.grad, want)
        # a caller may write to what it got
        leaf = logits.clone().requires_grad_()
        out = action_log_probs(leaf, actions)
        (out.log_prob * out.log_prob.detach().mul_(0.0).add_(1.0)).sum().backward()
        assert torch.isfinite(leaf.grad).all()


# ---------------------------------------------------------------------------- the policy they make up
def plain_policy(net, tokens, actions, state, resets, lengths, mask):
    """RecurrentActorNetwork.get_log_probs in torch, 64 bits, on the CPU; a loop over the steps."""
    p = {k: v.detach().double().cpu().requires_grad_() for k, v in net.named_parameters()}
    hidden = p["_head.weight"].shape[1]
    e = p["_embedding"][tokens.clamp(min=0)] * math.sqrt(hidden) * (tokens >= 0)[..., None]
    both = e @ p["_inputs.weight"].t() + p["_inputs.bias"]
    x, a = both[..., :hidden], torch.sigmoid(both[..., hidden:])
    h, outs = state, []
    for t in range(tokens.shape[1]):
        on = (t < lengths)[:, None]
        new = a[:, t] * torch.where(resets[:, t, None], torch.zeros_like(h), h) + (1 - a[:, t]) * x[:, t]
        h = torch.where(on, new, h)
        outs.append(torch.where(on, new, torch.zeros_like(new)))
    logits = torch.stack(outs, 1) @ p["_head.weight"].t() + p["_head.bias"]
    log_p = torch.log_softmax(logits.masked_fill(mask, float("-inf")), -1)
    prob = log_p.exp()
    entropy = -(prob * torch.where(mask, torch.zeros_like(log_p), log_p)).sum(-1)
    return p, logits, log_p.gather(-1, actions[..., None])[..., 0], entropy, h


@pytest.mark.parametrize("dtype,limit", [(torch.float32, 64 * 48 * O.U), (torch.bfloat16, 2.0 ** -5)], ids=["fp32", "bf16"])
@pytest.mark.parametrize("batch,time,actions", [(3, 70, 11), (2, 300, 900)])
def test_recurrent_actor_network(dtype, limit, batch, time, actions):
    """Forward and gradients of the three operators as one policy.  In fp32 each of four stages forwards
    and four backwards is off by at most (48 + 50) U of the norms it sums; in bf16 about eight roundings of
    2^-9 each stand in a row, and parameters are summed over all steps: both limits leave a factor of four
    for norms that cancel."""
    from pearl_amd import RecurrentActorNetwork
    torch.manual_seed(0)
    net = RecurrentActorNetwork(37, [48], actions).to(DEV, dtype)
    gen = gen_of(batch, time, actions)
    tokens = torch.randint(0, 37, (batch, time), generator=gen)
    lengths = torch.tensor([time, time - 9, 1][:batch])
    tokens[torch.arange(time)[None] >= lengths[:, None]] = -1
    acts = torch.randint(0, actions, (batch, time), generator=gen)
    resets = torch.rand(batch, time, generator=gen) < 0.03
    mask = torch.rand(batch, time, actions, generator=gen) < 0.2
    mask.scatter_(-1, acts[..., None], False)
    state = torch.randn(batch, 48, generator=gen)
    weight = torch.randn(batch, time, generator=gen) * (torch.arange(time)[None] < lengths[:, None])
    out, last = net.get_log_probs(tokens.to(DEV), acts.to(DEV), state.to(DEV), resets.to(DEV), lengths.to(DEV),
                                  mask.to(DEV), top=3)
    ((out.log_prob + 0.1 * out.entropy) * weight.to(DEV)).sum().backward()
    p, logits, lp, ent, h = plain_policy(net, tokens, acts, state.double(), resets, lengths, mask)
    ((lp + 0.1 * ent) * weight.double()).sum().backward()
    inside = weight != 0

    def off(got, want):
        return float((got.detach().double().cpu() - want.detach()).norm() / want.detach().norm())
    assert off(out.log_prob[inside.to(DEV)], lp[inside]) < limit and off(out.entropy[inside.to(DEV)], ent[inside]) < limit
    assert off(last, h) < limit
    for name, q in net.named_parameters():
        assert off(q.grad, p[name].grad) < limit, name


def test_recurrent_actor_network_acts_step_by_step_as_it_reads_histories():
    from pearl_amd import RecurrentActorNetwork
    torch.manual_seed(1)
    net = RecurrentActorNetwork(9, [40], 6).to(DEV)
    tokens = torch.randint(0, 9, (4, 50), device=DEV)
    resets = torch.rand(4, 50, device=DEV) < 0.1
    with torch.no_grad():
        logits, last = net(tokens, resets=resets)
    state = net.initial_state(4)
    for t in range(50):
        now, state = net.step(tokens[:, t], state, resets[:, t])
        torch.testing.assert_close(now, logits[:, t], rtol=0, atol=64 * 40 * O.U * float(logits.abs().max()))
    torch.testing.assert_close(state, last, rtol=0, atol=64 * 40 * O.U)
    with pytest.raises(NotImplementedError):
        net.linear_layers()


# ---------------------------------------------------------------------------- streams, graphs, devices
def a_run(s):
    """The three operators as a policy step uses them; `s` holds its inputs."""
    from pearl_amd import (action_log_probs, action_log_probs_grad, embed_tokens, embed_tokens_grad, gated_recurrence,
                           gated_recurrence_grad)
    e = embed_tokens(s["w"], s["tok"], scale=2.0)
    h, last, kept = gated_recurrence(e, s["g"], s["h0"], resets=s["r"], keep=True)
    logits = h @ s["head"]
    o = action_log_probs(logits, s["act"], top=5)
    dl = action_log_probs_grad(o, logits, s["act"], s["g_lp"], s["g_h"])
    dx, dg, d0 = gated_recurrence_grad(e, s["g"], kept, dl @ s["head_t"], resets=s["r"])
    dw = embed_tokens_grad(dx, s["tok"], s["w"].shape[0], scale=2.0)
    return [e, h, last, o.log_prob, o.entropy, o.top_actions, o.top_log_probs, dl, dx, dg, d0, dw]


def a_state(seed, b=2, t=700, d=48, vocab=300, width=5000):
    gen = gen_of(seed, 99)
    s = {"w": rnd(gen, vocab, d), "tok": torch.randint(0, vocab, (b, t), generator=gen).to(DEV), "g": rnd(gen, b, t, d) + 2,
         "h0": rnd(gen, b, d), "r": (torch.rand(b, t, generator=gen) < 0.02).to(DEV), "head": rnd(gen, d, width, scale=0.3),
         "act": torch.randint(0, width, (b, t), generator=gen).to(DEV), "g_lp": rnd(gen, b, t), "g_h": rnd(gen, b, t)}
    s["head_t"] = s["head"].t().contiguous()
    return s


def test_operators_on_two_streams_at_once():
    states = [a_state(k) for k in range(2)]
    want = [a_run(s) for s in states]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                got.append(a_run(s))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(g, w))


def test_operators_in_two_graphs_replayed_with_new_inputs():
    few = dict(b=1, t=900, d=24, vocab=100, width=20000)      # cut histories and rows: scratch in both graphs
    statics = [a_state(0, **few), a_state(1, **few)]
    a_run(statics[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in statics:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a_run(s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(a_run(s))
        graphs.append(g)
    for k in range(4):
        fresh = [a_state(10 + k, **few), a_state(20 + k, **few)]
        for s, f in zip(statics, fresh):
            for name in s:
                s[name].copy_(f[name])
        want = [a_run(f) for f in fresh]
        for g in (graphs if k % 2 else graphs[::-1]):
            g.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(got, w)), k


def test_acting_step_in_a_graph_advances_its_state_in_place():
    from pearl_amd import gated_recurrence, gated_recurrence_step
    gen = gen_of(61)
    xs, gs = rnd(gen, 3, 6, 21, dtype=torch.bfloat16), rnd(gen, 3, 6, 21, dtype=torch.bfloat16)
    x, g, state = xs[:, 0].clone(), gs[:, 0].clone(), torch.zeros(3, 21, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gated_recurrence_step(x, g, state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, _ = gated_recurrence_step(x, g, state, out_state=state)
    state.zero_()
    want, last = gated_recurrence(xs, gs)
    for t in range(6):
        x.copy_(xs[:, t])
        g.copy_(gs[:, t])
        graph.replay()
        torch.testing.assert_close(h.float(), want[:, t].float(), rtol=2.0 ** -7, atol=2.0 ** -14)
    torch.testing.assert_close(state, last, rtol=0, atol=100 * O.U * float(last.abs().max()))


def test_unknown_device_is_refused():
    from pearl_amd import _native as N
    w, tok, out = torch.randn(4, 4, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV), torch.empty(2, 4, device=DEV)
    rc = N.lib().pa_embed_tokens(w.data_ptr(), N.PA_F32, 4, 4, 4, tok.data_ptr(), N.PA_I64, 2, 1.0, out.data_ptr(), 1000, None)
    assert rc == N.PA_ERR_HIP and "1000" in N.last_error()
    assert torch.cuda.current_device() == 0


# ---------------------------------------------------------------------------- offsets behind 2^31 elements
def test_embed_tokens_behind_two_to_the_31st_element():
    from pearl_amd import embed_tokens, embed_tokens_grad
    vocab, dim = 2 ** 21 + 77, 1030
    w = torch.zeros(vocab, dim, dtype=torch.bfloat16, device=DEV)
    w[-3:] = torch.arange(3 * dim, device=DEV).view(3, dim).remainder(251).to(torch.bfloat16)
    tok = torch.tensor([vocab - 1, 0, vocab - 3, vocab - 1], device=DEV)
    out = embed_tokens(w, tok)
    assert torch.equal(out, w[tok]) and out[0].abs().sum() > 0
    d = torch.ones(4, dim, dtype=torch.bfloat16, device=DEV)
    dw = embed_tokens_grad(d, tok, vocab)
    assert (dw[-1] == 2).all() and (dw[-2] == 0).all() and (dw[-3] == 1).all() and (dw[0] == 1).all()
    assert float(dw[1:-3].abs().max()) == 0


def test_gated_recurrence_behind_two_to_the_31st_element():
    from pearl_amd import gated_recurrence, gated_recurrence_grad
    t, d = 2 ** 21 + 1000, 1030
    x = torch.empty(1, t, d, dtype=torch.bfloat16, device=DEV).normal_()
    g = torch.empty(1, t, d, dtype=torch.bfloat16, device=DEV).normal_()
    h, last, kept = gated_recurrence(x, g, keep=True)
    cut = t - 500
    _, middle = gated_recurrence(x[:, cut - 2000:cut], g[:, cut - 2000:cut])     # gates near 1/2: far states do not matter
    h2, last2, kept2 = gated_recurrence(x[:, cut:], g[:, cut:], middle, keep=True)
    torch.testing.assert_close(last, last2, rtol=0, atol=200 * O.U * 4)
    torch.testing.assert_close(h[:, cut:].float(), h2.float(), rtol=2.0 ** -7, atol=2.0 ** -12)
    d_h = torch.empty(1, t, d, dtype=torch.bfloat16, device=DEV).normal_()
    a = gated_recurrence_grad(x, g, kept, d_h)
    b = gated_recurrence_grad(x[:, cut:], g[:, cut:], kept2, d_h[:, cut:])
    for k in (0, 1):
        torch.testing.assert_close(a[k][:, cut:].float(), b[k].float(), rtol=2.0 ** -7, atol=2.0 ** -10)


def test_action_log_probs_behind_two_to_the_31st_element():
    from pearl_amd import action_log_probs, action_log_probs_grad
    rows, width = 66000, 32771
    logits = torch.empty(rows, width, dtype=torch.bfloat16, device=DEV).normal_()
    actions = torch.randint(0, width, (rows,), device=DEV)
    o = action_log_probs(logits, actions, top=3)
    few = action_log_probs(logits[-600:], actions[-600:], top=3)
    assert torch.equal(o.log_prob[-600:], few.log_prob) and torch.equal(o.entropy[-600:], few.entropy)
    assert torch.equal(o.top_actions[-600:], few.top_actions)
    g_lp, g_h = torch.randn(rows, device=DEV), torch.randn(rows, device=DEV)
    d = action_log_probs_grad(o, logits, actions, g_lp, g_h)
    assert torch.equal(d[-600:], action_log_probs_grad(few, logits[-600:], actions[-600:], g_lp[-600:], g_h[-600:]))
    want = O.log_probs(np64(logits[-2:]), actions[-2:].cpu().numpy(), None, 1.0, 3, np64(g_lp[-2:]), np64(g_h[-2:]))
    O.check(o.log_prob[-2:], *want["log_prob"], torch.float32, "log_prob")
    O.check(d[-2:], *want["d_logits"], torch.bfloat16, "d_logits")
