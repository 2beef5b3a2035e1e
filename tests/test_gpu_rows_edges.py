"""GPU: the row operators where their arithmetic ends, against oracle/rows.py in float64.  The tolerances are those of test_gpu_rows.py."""
import math

import numpy as np
import pytest
import torch

from oracle import rows as orow
from test_gpu_rows import U, check_distill, check_drawn, cuda, distill_case, host, rows_of, sum_error

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


# ------------------------------------------------------------------------------------------------ drawing
@pytest.mark.parametrize("dtype,V", [(torch.float32, 48), (torch.float32, 1000), (torch.float32, 9000), (torch.bfloat16, 9000), (torch.bfloat16, 70000), (torch.float16, 70000)])
@pytest.mark.parametrize("k", [0, 600])
def test_a_row_s_top_p_of_nothing_keeps_the_first_token(dtype, V, k):
    """Flat rows: more tokens of one value than a bin's list (fp32) or a counter (16 bits, 70,000 tokens) holds."""
    from mucon_amd import ops

    x = rows_of("flat", 4, V, dtype, 1)
    x[1] = rows_of("normal", 1, V, dtype, 2)[0]
    x[2, V // 2] = 1.5
    x[3, :7] = -math.inf
    p = torch.tensor([0.0, -1.0, -math.inf, 0.0])
    u = torch.tensor([0.0, 0.5, 0.999, 0.7])
    for T in (1.0, 50.0):
        for m in (0.0, 0.5):
            token, logp = ops.sample_logits(*cuda(x, u), T, k, p.cuda(), m)
            assert token.tolist() == [int(orow.order(r)[0]) for r in host(x)]
            assert logp.tolist() == [0.0] * 4


@pytest.mark.parametrize("dtype,V", [(torch.float32, 9000), (torch.float32, 4097), (torch.bfloat16, 9000), (torch.bfloat16, 200000)])
@pytest.mark.parametrize("T", [1e30, 1.1e37, 3e37, 3.4e38, math.inf])
@pytest.mark.parametrize("k", [600, 5000, 0])
def test_draws_at_temperatures_near_the_end_of_fp32(dtype, V, T, k):
    """Few tokens above -inf, fewer than top_k; all of them are alike at these temperatures: weights within 2^-90 of 1.  (70,000 and more tokens of one 16-bit value
    run over its counter: -inf is counted apart, so the last size has that many finite ones.)"""
    from mucon_amd import ops

    x = torch.full((5, V), -math.inf)
    g = torch.Generator().manual_seed(3)
    for r, n in enumerate((20, 1, 599, 600, 601)):
        x[r, torch.randperm(V, generator=g)[:n]] = torch.randn(n, generator=g)
    if V > 65536:
        x[4, 1000:80000] = 0.5
    x = x.to(dtype)
    u = torch.tensor([0.6, 0.9, 0.999, 0.37, 0.99])
    token, logp = ops.sample_logits(*cuda(x, u), torch.full((5,), T).cuda(), k)
    for r in range(5):
        finite = int((x[r] > -math.inf).sum())
        n = min(finite, k) if k else finite
        at = min(int(np.float64(u[r]) * n), n - 1)      # the sums are whole numbers: the first above u n
        assert int(token[r]) == int(orow.order(host(x)[r])[at]), (r, n)
        assert abs(float(logp[r]) + math.log(n)) <= U * math.log(n) + 1e-11


def test_draws_of_logits_at_the_end_of_fp32():
    """A bin's borders in the row's units overflow where the logits themselves are near the largest of fp32."""
    from mucon_amd import ops

    V = 9000
    x = torch.full((3, V), -3.0e38)
    x[0, 17], x[0, 5] = 3.0e38, 2.9e38
    x[1, ::2] = 3.0e38
    x[2, 8000:] = 1.0e38
    u = torch.tensor([0.6, 0.9, 0.5])
    for T in (1e36, 3e37, 3e38):
        for k, p in ((0, 1.0), (600, 1.0), (0, 0.9), (5000, 0.9)):
            token, logp = ops.sample_logits(*cuda(x, u), torch.full((3,), T).cuda(), k, p)
            check_drawn(token.cpu(), logp.cpu(), host(x), u, (np.float32(T).item(), k, np.float32(p).item(), 0.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [48, 200, 900, 3000, 9000, 70000])
def test_few_tokens_allowed_and_more_asked_for(V, dtype):
    """Rows of which 20 tokens are above -inf, with top_k and k beyond that: all of them, then (of top_logits) the masked ones by their index."""
    from mucon_amd import ops

    g = torch.Generator().manual_seed(V)
    x = torch.full((4, V), -math.inf)
    for r in range(4):
        x[r, torch.randperm(V, generator=g)[:20]] = torch.randn(20, generator=g)
    x = x.to(dtype)
    for k in (19, 20, 21, min(V, 50), min(V, 1000)):
        top = ops.top_logits(x.cuda(), k, 0.8)
        values, index, lse = orow.top(host(x), k, 0.8)
        assert np.array_equal(top.index.cpu().numpy(), index) and np.array_equal(host(top.values), values)
        assert np.allclose(top.lse.cpu().numpy(), lse, rtol=U, atol=sum_error(V))
    u = torch.tensor([0.0, 0.3, 0.7, 1.0 - 2.0 ** -24])
    for k in (19, 20, 21, 50, 1000, 5000):
        for p, m in ((1.0, 0.0), (0.8, 0.0), (1.0, 0.2), (0.9, 0.05)):
            token, logp = ops.sample_logits(*cuda(x, u), 0.8, k, p, m)
            check_drawn(token.cpu(), logp.cpu(), host(x), u, (np.float32(0.8).item(), k, np.float32(p).item(), np.float32(m).item()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["flat", "ties", "normal"])
@pytest.mark.parametrize("V", [48, 200, 900, 3000, 9000, 70000])
def test_rows_of_their_own_parameters_in_every_type(V, kind, dtype):
    from mucon_amd import ops

    if V == 70000 and kind == "ties":
        pytest.skip("as 9,000")
    rows = 16
    x = rows_of(kind, rows, V, dtype, 7)
    x[3, V // 3:] = -math.inf
    g = torch.Generator().manual_seed(V)
    T = torch.rand(rows, generator=g) * 2 + 0.3
    k = torch.randint(0, 2 * min(V, 1500), (rows,), generator=g).to(torch.int32)
    p, m = torch.rand(rows, generator=g) * 1.3, torch.rand(rows, generator=g) * 0.3
    T[0], k[1], p[2], m[4], p[5], k[6] = 0.0, 0, 0.0, 1.0, -0.5, 1
    u = torch.rand(rows, generator=g)
    token, logp = ops.sample_logits(*cuda(x, u), *cuda(T, k, p, m))
    check_drawn(token.cpu(), logp.cpu(), host(x), u, (T, torch.where(k >= V, torch.zeros_like(k), k), p, m))


# ------------------------------------------------------------------------------------------------ distillation
def far_case(V, dtype, T, seed, levels, rest_mass=0.5, rows=4):
    """Unlisted student logits within half a unit of 0, listed ones at `levels` (exact in every type); the teacher leaves `rest_mass` to the unlisted tokens."""
    g = torch.Generator().manual_seed(seed)
    s = torch.randint(-8, 9, (rows, V), generator=g).float() / 16.0
    K = len(levels)
    index = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(rows)]).to(torch.int32)
    s.scatter_(1, index.long(), torch.tensor(levels).expand(rows, K))
    values = torch.randint(-4, 5, (rows, K), generator=g).float() * (T / 4.0)
    lse = (torch.logsumexp(values.double() / T, 1) - math.log(1.0 - rest_mass)).float()
    return s.to(dtype), values, index, lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [7, 48, 64, 65, 900, 9000, 40000, 131072])
@pytest.mark.parametrize("T,levels", [(0.1, [6.0, 12.0]), (0.1, [9.0, 9.0, 9.0]), (1.0, [95.0, 88.0]), (0.5, [-60.0, -100.0, -60.0]), (0.05, [8.0, 16.0, 24.0])])
def test_distill_students_far_from_their_teacher(V, dtype, T, levels):
    """The unlisted tokens' mass is e^-60 to e^-480 of the row's, below the smallest fp32: the rest term and its gradient are those of the definition, and finite (in the
    fourth case it is the listed tokens' mass that is small)."""
    from mucon_amd import ops

    s, values, index, lse = far_case(V, dtype, T, V, levels)
    leaf = s.cuda().requires_grad_(True)
    d = cuda(values, index, lse)
    for reduction in ("none", "sum"):
        loss = ops.distill_loss(leaf, *d, temperature=T, reduction=reduction)
        grad, = torch.autograd.grad(loss.sum(), leaf)
        assert bool(grad.isfinite().all()) and bool(loss.isfinite().all())
        check_distill(loss.detach(), grad, s, values, index, lse, None, T, reduction)
        loss, grad = ops.distill_loss_and_grad(s.cuda(), *d, temperature=T, reduction=reduction, grad_scale=2.0)
        check_distill(loss, grad, s, values, index, lse, None, T, reduction, torch.full((4,), 2.0) if reduction == "none" else 2.0)


@pytest.mark.parametrize("V", [48, 900, 40000, 131072])
def test_distill_of_a_far_row_under_a_loss_scale(V):
    """A scaled loss, as for 16-bit gradients: the gradient of the definition times the scale."""
    from mucon_amd import ops

    T, scale = 0.1, 65536.0
    for levels in ([8.25, 8.5], [8.5, 8.75], [8.75, 8.75]):      # e^-82 .. e^-88: around the smallest fp32
        s, values, index, lse = far_case(V, torch.float32, T, V, levels)
        leaf = s.cuda().requires_grad_(True)
        d = cuda(values, index, lse)
        loss = ops.distill_loss(leaf, *d, temperature=T, reduction="sum")
        grad, = torch.autograd.grad(loss, leaf, torch.tensor(scale).cuda())
        check_distill(loss.detach(), grad, s, values, index, lse, None, T, "sum", scale)
        _, grad = ops.distill_loss_and_grad(s.cuda(), *d, temperature=T, reduction="sum", grad_scale=scale)
        check_distill(loss.detach(), grad, s, values, index, lse, None, T, "sum", scale)


@pytest.mark.parametrize("V", [48, 900, 40000, 131072])
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_far_rows_whose_unlisted_tokens_rise(V, dtype):
    """Unlisted logits that grow along the row, and listed ones between and above them, some listed twice, one of them -inf: the running maximum moves with every step."""
    from mucon_amd import ops

    T = 0.25
    s = (torch.arange(V) * 32 // V).float().repeat(3, 1)
    index = torch.tensor([[V - 1, 0, 3, 0], [V // 2, V // 2 + 1, -1, V // 2], [1, 2, 3, V]], dtype=torch.int32)
    s[0, 0], s[0, 3], s[0, V - 1] = 80.0, 40.0, -math.inf
    s[1, V // 2] = 64.0
    s[2, 1:4] = torch.tensor([-40.0, 16.0, 120.0])
    s = s.to(dtype)
    values = torch.tensor([[-math.inf, 1.0, 0.0, 0.5], [0.0, 0.25, 9.0, 0.0], [0.5, 0.0, 0.25, 0.0]])
    lse = torch.tensor([5.5, 3.0, 4.0])
    leaf = s.cuda().requires_grad_(True)
    d = cuda(values, index, lse)
    loss = ops.distill_loss(leaf, *d, temperature=T, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), leaf)
    check_distill(loss.detach(), grad, s, values, index, lse, None, T, "none")
    loss, grad = ops.distill_loss_and_grad(s.cuda(), *d, temperature=T, reduction="none")
    check_distill(loss, grad, s, values, index, lse, None, T, "none")


@pytest.mark.parametrize("V", [7, 48, 900, 40000])
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_where_every_unlisted_token_is_masked(V, dtype):
    """A vocabulary masked down to the listed tokens, whose logits lie far below, around and above 0: there is no rest term, and no gradient elsewhere."""
    from mucon_amd import ops

    for T in (0.004, 1.0):
        s, values, index, lse = far_case(V, dtype, T, 3, [0.0, 0.25, 0.5])
        for shift in (-60.0, 0.0, 60.0):
            x = torch.full_like(s, -math.inf).scatter(1, index.long(), (s.float().gather(1, index.long()) + shift).to(dtype))
            leaf = x.cuda().requires_grad_(True)
            loss = ops.distill_loss(leaf, *cuda(values, index, lse), temperature=T, reduction="none")
            grad, = torch.autograd.grad(loss.sum(), leaf)
            check_distill(loss.detach(), grad, x, values, index, lse, None, T, "none")
            loss, grad = ops.distill_loss_and_grad(x.cuda(), *cuda(values, index, lse), temperature=T, reduction="none")
            check_distill(loss, grad, x, values, index, lse, None, T, "none")
            assert not grad[x.isneginf().cuda()].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_distill_with_a_rest_at_a_low_temperature_and_far_from_zero(dtype):
    """Logits around 60 at temperature 1/20 with the teacher's log-sum-exp given: near 1,200, where its own step in fp32 is 2^-13, which enters 1 - sum p as it is given."""
    from mucon_amd import ops

    for V in (48, 900, 40000):
        g = torch.Generator().manual_seed(6)
        s = (60.0 + 0.25 * torch.randint(-6, 7, (5, V), generator=g)).to(dtype)        # (exact in every type)
        t = (60.0 + 0.25 * torch.randint(-6, 7, (5, V), generator=g)).to(dtype)
        values, index = t.float().topk(5, dim=1)
        lse = (torch.logsumexp(t.double() / 0.05, 1)).float()
        values, index = values.to(dtype), index.to(torch.int32)
        leaf = s.cuda().requires_grad_(True)
        loss = ops.distill_loss(leaf, *cuda(values, index, lse), temperature=0.05, reduction="sum")
        grad, = torch.autograd.grad(loss, leaf)
        check_distill(loss.detach(), grad, s, values, index, lse, None, 0.05, "sum")
        loss, grad = ops.distill_loss_and_grad(s.cuda(), *cuda(values, index, lse), temperature=0.05, reduction="sum")
        check_distill(loss, grad, s, values, index, lse, None, 0.05, "sum")


def plain_distill(s, values, index, lse, T):
    """The rows' losses in torch operations: exponentials in fp32, sums and the few listed entries in 64 bits."""
    at, top = index.long(), s.detach().max(dim=1, keepdim=True).values
    e = ((s - top) / T).exp()
    log_total = e.sum(dim=1, dtype=torch.float64).log()
    log_q = (s.gather(1, at).double() - top.double()) / T - log_total[:, None]
    log_p = values.double() / T - lse.double()[:, None]
    p = log_p.exp()
    rest = 1.0 - p.sum(dim=1)
    outside = torch.where(torch.zeros_like(e).scatter_(1, at, 1.0) > 0, torch.zeros_like(e), e).sum(dim=1, dtype=torch.float64)
    return ((p * (log_p - log_q)).sum(dim=1) + rest * (rest.log() - outside.log() + log_total)) * T * T


@pytest.mark.parametrize("rows,V", [(512, 49), (256, 300), (128, 3000), (64, 20001), (48, 50001)])
@pytest.mark.parametrize("T", [1.0, 2.0, 1.3, 0.7])
def test_distill_in_fp32_is_as_near_the_definition_as_the_plain_form(rows, V, T):
    """The root mean square of the rows' losses' errors and of the gradient's elements', each against 64 bits, are at most those of the same formula in torch's fp32 operations: a
    constant of the exponent in one fp32 number (T = 1, 2), or coefficients in fp32, show here as a bias.  (A tenth more for chance: both hold the final rounding, whose mean square over
    48 losses varies by 1 / sqrt(5 / 4 x 48) = 0.13, a root of 0.065.)"""
    from mucon_amd import ops

    s, values, index, lse, _ = distill_case(rows, V, 16, torch.float32, torch.float32, True, False, V, T)
    s, values, index, lse = cuda(s, values, index, lse)
    exact = s.double().requires_grad_(True)
    log_q = torch.log_softmax(exact / T, 1)
    log_p = values.double() / T - lse.double()[:, None]
    p = log_p.exp()
    rest = 1.0 - p.sum(1)
    unlisted = torch.ones_like(log_q).scatter(1, index.long(), 0.0)
    want = ((p * (log_p - log_q.gather(1, index.long()))).sum(1) + rest * (rest.log() - (unlisted * log_q.exp()).sum(1).log())) * T * T
    want_grad, = torch.autograd.grad(want.mean(), exact)

    def errors(loss, grad):
        return [float((a.double() - b).norm() / b.norm()) for a, b in ((loss, want.detach()), (grad, want_grad))]

    plain = s.clone().requires_grad_(True)
    of_plain = errors(plain_distill(plain, values, index, lse, T).detach().float(), torch.autograd.grad(plain_distill(plain, values, index, lse, T).mean().float(), plain)[0])
    leaf = s.clone().requires_grad_(True)
    loss = ops.distill_loss(leaf, values, index, lse, temperature=T, reduction="none").detach()
    for grad in (torch.autograd.grad(ops.distill_loss(leaf, values, index, lse, temperature=T), leaf)[0], ops.distill_loss_and_grad(s, values, index, lse, temperature=T)[1]):
        for mine, theirs in zip(errors(loss, grad), of_plain):
            assert mine <= 1.1 * theirs, (errors(loss, grad), of_plain)


@pytest.mark.parametrize("rows,V,K", [(40, 49, 4), (9, 300, 16), (5, 4000, 40), (3, 20001, 64), (2, 131072, 64), (1, 262144, 1024)])
@pytest.mark.parametrize("T", [1.0, 0.6])
def test_distill_gradients_in_fp32_element_by_element(rows, V, K, T):
    """An unlisted token's weight is exp2 of an exponent of t: the difference and the product round once each (2 t u ln 2 of the weight), exp2 to a step (2 u), the last product and the
    result once (2 u).  The row's sum has that of its mean exponent, at most log2 V, and three roundings of a vector's; it enters every element in its share.  A listed token's own
    terms are 64-bit."""
    from mucon_amd import ops

    s, values, index, lse, _ = distill_case(rows, V, K, torch.float32, torch.float32, True, False, V + K, T)
    want = orow.distill(s, values, index, lse, T, None, "none")[1]
    q = torch.softmax(s.double() / T, 1)
    listed = torch.zeros_like(q).scatter(1, index.long(), 1.0) > 0
    mo = torch.where(listed, torch.full_like(s, -math.inf), s).max(1, keepdim=True).values.double()
    p = torch.exp(values.double() / T - lse.double()[:, None])
    rest = (1.0 - p.sum(1, keepdim=True)).clamp(min=0)
    share = T * (q + torch.where(listed, 0.0, rest * q / (q * ~listed).sum(1, keepdim=True)))
    t = (mo - s.double()) / T / math.log(2)
    of_sum = (2 * math.log(2) * math.log2(V) + 2 + 3) * U
    bound = share * (of_sum + torch.where(listed, 0.0, (2 * math.log(2) * t + 4) * U)) + U * want.abs() + 1e-14
    leaf = s.cuda().requires_grad_(True)
    d = cuda(values, index, lse)
    for grad in (torch.autograd.grad(ops.distill_loss(leaf, *d, temperature=T, reduction="sum"), leaf)[0], ops.distill_loss_and_grad(s.cuda(), *d, temperature=T, reduction="sum")[1]):
        err = (grad.double().cpu() - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())


# ------------------------------------------------------------------------------------------------ calls
def test_the_operators_called_by_name():
    from mucon_amd import ops

    s, values, index, lse = far_case(300, torch.bfloat16, 1.0, 1, [1.0, 2.0, 0.5])
    s, values, index, lse, u = cuda(s, values, index, lse, torch.rand(4))
    assert all(torch.equal(a, b) for a, b in zip(ops.top_logits(logits=s, k=5), ops.top_logits(s, 5)))
    assert all(torch.equal(a, b) for a, b in zip(ops.sample_logits(uniform=u, logits=s), ops.sample_logits(s, u)))
    listed = dict(teacher_values=values, teacher_index=index, teacher_lse=lse)
    assert torch.equal(ops.distill_loss(student=s, **listed), ops.distill_loss(s, values, index, lse))
    assert all(torch.equal(a, b) for a, b in zip(ops.distill_loss_and_grad(student=s, **listed), ops.distill_loss_and_grad(s, values, index, lse)))


# ------------------------------------------------------------------------------------------------ in the model
def a_model(hidden):
    from mucon_amd.config import get_cfg_defaults, update_config
    from mucon_amd.mucon.models import create_model
    from test_gpu_model import seeded_value

    over = ["model.fs.encoder.hidden_size", str(hidden), "model.fs.decoder.hidden_size", str(hidden)]
    model = create_model(update_config(get_cfg_defaults(), [], [over]), num_classes=48, max_decoding_steps=31, input_feature_size=2048)
    with torch.no_grad():
        for name, p in model.named_parameters():
            p.copy_(torch.from_numpy(seeded_value(name, p.shape).astype(np.float32)))
    return model.cuda().eval()


@pytest.mark.parametrize("hidden", [128, 64])
def test_a_transcript_drawn_by_the_module_decoder(hidden, monkeypatch):
    """native_decoder = False, and a decoder narrower than the native one's: the module's steps, with temperature 0 its greedy words, with uniforms the row oracle's
    draws from its rows over the words before."""
    from mucon_amd import ops
    from test_gpu_model import make_batch

    model, batch = a_model(hidden), make_batch(640, 5).to("cuda")
    model.native_decoder = hidden != 128
    u = torch.rand(31, generator=torch.Generator().manual_seed(3))

    def no_native(*args, **kw):
        raise AssertionError("the native decoder was called")

    monkeypatch.setattr(ops, "decoder_forward", no_native)
    model.set_teacher_forcing(False)
    with torch.no_grad():
        greedy = model.forward(batch).transcript.argmax(dim=1).tolist()
    words, logp = model.sample_transcript(batch, u.cuda(), temperature=0.0)
    assert words == greedy and not logp.any()
    words, logp = model.sample_transcript(batch, u.cuda(), temperature=1.5, top_p=0.95)
    assert len(words) == len(logp) and (words[-1] == model.EOS_token_id or len(words) == 31)
    model.set_teacher_forcing(True)
    with torch.no_grad():
        given = torch.tensor([49] + words[:-1]).cuda()
        rows, _ = model.sequence_generation_forward(model.temporal_modeling_forward(input=batch.feats), len(words), given, given)
    check_drawn(words, logp.cpu(), host(torch.cat(rows)), u, (1.5, 0, np.float32(0.95).item(), 0.0))
    if hidden == 128:
        monkeypatch.undo()
        model.native_decoder = True
        again, _ = model.sample_transcript(batch, u.cuda(), temperature=1.5, top_p=0.95)
        assert again == words      # (the rows agree to fp32, the uniforms are not at a border)


def test_what_is_drawn_behind_the_end_mark_does_not_count(monkeypatch):
    """A row without a distribution (token -1) is an error in front of the end mark, nothing behind it."""
    from mucon_amd import ops
    from test_gpu_model import make_batch

    model, batch = a_model(128), make_batch(640, 5).to("cuda")
    for drawn, words in (([3, 7, 48, -1, 5], [3, 7, 48]), ([3, -1, 48, 1, 5], None), ([3, 7, 1, 1, -1], None)):
        left = iter(drawn)
        monkeypatch.setattr(ops, "sample_logits", lambda *a: (torch.tensor(next(left), device="cuda"), torch.tensor(-0.5, device="cuda")))
        if words is None:
            with pytest.raises(RuntimeError, match="not finite"):
                model.sample_transcript(batch, torch.rand(5).cuda())
        else:
            got, logp = model.sample_transcript(batch, torch.rand(5).cuda())
            assert got == words and len(logp) == len(words)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [48, 200, 900, 9000, 40000])
@pytest.mark.parametrize("T", [1e-30, 1e-6, 1e4, 1e30])      # (a gradient of T p: 65,504 is the largest of fp16)
def test_the_ends_of_the_temperatures(V, dtype, T):
    """Masked rows at the smallest and largest temperatures: one token or all of them alike."""
    from mucon_amd import ops

    x = rows_of("masked", 3, V, dtype, 4)
    top = ops.top_logits(x.cuda(), 2, T)
    values, index, lse = orow.top(host(x), 2, T)
    assert np.array_equal(top.index.cpu().numpy(), index)
    assert np.allclose(top.lse.cpu().numpy(), lse, rtol=U, atol=sum_error(V))
    if T > 1e18:      # (T^2 L leaves fp32)
        return
    for given in (None, torch.from_numpy(np.float32(lse)) if T > 1 else None):      # (at the small ones a step of the log-sum-exp in fp32 is 1 and more: no distribution)
        leaf = x.cuda().requires_grad_(True)
        values = torch.from_numpy(host(top.values))
        values[0] = values[0, 0]      # (the largest twice: half a probability each)
        loss = ops.distill_loss(leaf, *cuda(values, top.index, given), temperature=T, reduction="none")
        grad, = torch.autograd.grad(loss.sum(), leaf)
        check_distill(loss.detach(), grad, x, values, top.index.cpu(), given, None, T, "none")
