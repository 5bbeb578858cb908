"""Log probabilities with entropy and alternatives, and distillation from top logits, against 64-bit definitions.

The CPU tests check the reference forms (values, gradients by differences,
refusals); the GPU tests compare the kernels with the reference forms in
fp64 on the same inputs.

Tolerances. A log probability is ln 2 ((z - m) c - log2 S): the product
carries three fp32 roundings (2^-24 each, relative), the sum S of exponentials
accurate to 2^-22 adds 2^-22 to its logarithm, and the last subtraction rounds
once more, so an error of |log p| 2^-22 + 2^-20 is allowed. The entropy adds
sum p log p whose terms each carry the error of p (2^-22, and 2^-24 |x| of the
exponent) and of the logarithm: (H + log V) 2^-20 + 2^-19. Gradients are sums
of two products of p with rows' factors of size G: p is off by 2^-22 and by
2^-24 times an exponent below 128 where it matters (p > 2^-128), relative, so
G 2^-17 covers p <= 1, plus half a step of the logits' type.
"""

import math

import pytest
import torch

from koochak_b200.ops import functional as kf

DEV = "cuda"
gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IGNORE = -100


@pytest.fixture(autouse=True)
def _status_clean(request):
    yield
    if "gpu" in request.keywords and torch.cuda.is_available():
        from koochak_b200.ops import check_status

        torch.cuda.synchronize()
        check_status()


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _logits(rows, vocab, dtype, layout="padded", seed=0, device=DEV, sigma=2.0):
    """[rows, vocab] logits with some likely tokens; ``layout`` decides strides and alignment."""

    gen = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, vocab, generator=gen) * sigma
    n = min(8, vocab)
    ids = torch.stack([torch.randperm(vocab, generator=gen)[:n] for _ in range(rows)]) if rows else \
        torch.zeros(0, n, dtype=torch.int64)
    z.scatter_add_(1, ids, torch.full((rows, n), 6.0))
    z = z.to(device, dtype)
    if layout == "contiguous":
        return z
    if layout == "padded":
        ld = (vocab + 63) // 64 * 64
        buf = torch.full((rows, ld), math.nan, device=device, dtype=dtype)
    elif layout == "offset":  # rows start off every 16-byte boundary, by another distance each
        buf = torch.full((rows, vocab + 5), math.nan, device=device, dtype=dtype)[:, 1:]
    elif layout == "columns":  # inner stride is not one
        buf = torch.full((vocab, rows), math.nan, device=device, dtype=dtype).t()
    else:
        raise AssertionError(layout)
    buf = buf[:, :vocab]
    buf.copy_(z)
    return buf


def _close(got, want, tol, what):
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape, what
    same = (got == want) | (got.isnan() & want.isnan())
    err = torch.where(same, 0.0, (got - want).abs())
    bad = ~(err <= (tol.double().cpu() if isinstance(tol, torch.Tensor) else tol))
    assert not bad.any(), f"{what}: {bad.sum()} off, {got[bad][:4]} for {want[bad][:4]}"


def _logprob_tol(want):
    return torch.nan_to_num(want.abs(), nan=0.0, posinf=0.0) * 2.0**-22 + 2.0**-20


def _check_logprobs(z, tokens, top_k=0, temperature=1.0, grads=True, seed=0):
    vocab = z.shape[-1]
    rows = z.numel() // vocab
    z = z.detach().requires_grad_(grads)
    res = kf.token_logprobs(z, tokens, top_k=top_k, temperature=temperature, ignore_index=IGNORE)
    ref_z = z.detach().cpu().double().reshape(rows, vocab).requires_grad_(grads)
    flat = None if tokens is None else tokens.cpu().reshape(-1)
    logp, ent, tlp, tid = kf.token_logprobs_ref(ref_z, flat, top_k=top_k, temperature=temperature,
                                                ignore_index=IGNORE)
    lead = z.shape[:-1]
    assert res.entropy.shape == lead and res.entropy.dtype == torch.float32
    if tokens is None:
        assert res.logprobs is None
    else:
        _close(res.logprobs.detach().reshape(-1), logp.detach(), _logprob_tol(logp.detach()), "logprobs")
    tol = (ent.detach().nan_to_num(0.0).abs() + math.log(vocab)) * 2.0**-20 + 2.0**-19
    _close(res.entropy.detach().reshape(-1), ent.detach(), tol, "entropy")
    if top_k:
        assert torch.equal(res.top_ids.cpu().reshape(rows, top_k), tid)
        _close(res.top_logprobs.reshape(rows, top_k), tlp, _logprob_tol(tlp), "top_logprobs")
    if not grads:
        return res
    gen = torch.Generator().manual_seed(seed + 1)
    dlp, dh = torch.randn(rows, generator=gen), torch.randn(rows, generator=gen) * 0.3
    outs, gs = [res.entropy.reshape(-1)], [dh.to(z.device)]
    ref_outs, ref_gs = [ent], [dh.double()]
    if tokens is not None:
        outs, gs = outs + [res.logprobs.reshape(-1)], gs + [dlp.to(z.device)]
        ref_outs, ref_gs = ref_outs + [logp], ref_gs + [dlp.double()]
    (dz,) = torch.autograd.grad(outs, z, gs)
    (want,) = torch.autograd.grad(ref_outs, ref_z, ref_gs)
    assert dz.shape == z.shape and dz.dtype == z.dtype
    size = (dlp.abs() + dh.abs() * (ent.detach().nan_to_num(0.0) + 1.0)).double() / temperature
    tol = size[:, None] * 2.0**-17 + want.nan_to_num(0.0).abs() * _half_step(z.dtype) * (1 + 2.0**-10)
    tol = tol + torch.finfo(z.dtype).tiny * _half_step(z.dtype) * 2
    _close(dz.reshape(rows, vocab), want, tol, "dlogits")
    return res


def _tokens(rows, vocab, device=DEV, seed=0, ignored=True):
    gen = torch.Generator().manual_seed(seed + 7)
    t = torch.randint(0, vocab, (rows,), generator=gen)
    if ignored and rows > 2:
        t[::5] = IGNORE
    return t.to(device)


# ------------------------------------------------------------------- CPU


@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_reference_logprobs_and_gradient_by_differences(temperature):
    torch.manual_seed(0)
    z = torch.randn(3, 11, dtype=torch.float64, requires_grad=True)
    tokens = torch.tensor([2, IGNORE, 10])

    def f(x):
        lp, ent, _, _ = kf.token_logprobs_ref(x, tokens, temperature=temperature, ignore_index=IGNORE)
        return lp, ent

    p = torch.softmax(z / temperature, -1)
    lp, ent = f(z)
    assert torch.allclose(lp[0], p[0, 2].log()) and lp[1] == 0 and ent[1] == 0
    assert torch.allclose(ent[2], -(p[2] * p[2].log()).sum())
    assert torch.autograd.gradcheck(f, (z,))
    (g,) = torch.autograd.grad((lp[0] * 0.5 + ent[0] * 0.25), z)
    hot = torch.zeros(11, dtype=torch.float64)
    hot[2] = 1
    want = (0.5 * (hot - p[0]) - 0.25 * p[0] * (p[0].log() + ent[0])) / temperature
    assert torch.allclose(g[0], want) and not g[1].any()


@pytest.mark.parametrize("tail", [False, True])
def test_reference_distillation_and_gradient_by_differences(tail):
    torch.manual_seed(1)
    z = torch.randn(4, 9, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[1, 5, 8], [0, -1, 3], [-1, -1, 99], [2, 2, 4]])
    t = torch.log_softmax(torch.randn(4, 4, dtype=torch.float64), -1)[:, :3]
    temperature = 1.5

    def f(x):
        return kf.topk_distillation_ref(x, ids, t, temperature=temperature, tail=tail)

    loss = f(z)
    assert loss[2] == 0 and torch.autograd.gradcheck(f, (z,))
    p = torch.softmax(z.detach() / temperature, -1)
    q = t[0].exp() if tail else torch.softmax(t[0] / temperature, -1)
    want = (q * (q.log() - p[0, ids[0]].log())).sum()
    if tail:
        rest, p_rest = 1 - q.sum(), 1 - p[0, ids[0]].sum()
        want = want + rest * (rest / p_rest).log()
    assert torch.allclose(loss[0], want)
    (g,) = torch.autograd.grad(loss[0], z)
    dz = p[0].clone() if tail else p[0] * q.sum()
    dz[ids[0]] -= q
    if tail:
        off = torch.ones(9, dtype=torch.bool)
        off[ids[0]] = False
        dz[off] -= rest * p[0][off] / p_rest
    assert torch.allclose(g[0], dz / temperature)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("far", [1e3, 1e8, 1e30])
def test_reference_rest_far_below_the_list(dtype, far):
    """The gradient off the list is the rest's share, softmax over the tokens off the list, however far they are. The
    listed token has all of the student's mass, so its own gradient is the rest's probability."""

    gen = torch.Generator().manual_seed(9)
    z = torch.randn(2, 50, generator=gen, dtype=dtype)
    z[:, 7] = far
    z.requires_grad_()
    t = torch.tensor([[0.75]] * 2, dtype=dtype).log()
    loss = kf.topk_distillation_ref(z, torch.tensor([[7]] * 2), t, temperature=2.0, tail=True)
    (dz,) = torch.autograd.grad(loss.sum(), z)
    share = torch.softmax(torch.cat([z[:, :7], z[:, 8:]], 1).detach().double() / 2.0, 1)
    want = -0.25 * torch.cat([share[:, :7], torch.full((2, 1), -1.0), share[:, 7:]], 1) / 2.0
    # a few roundings of a share, a product and a quotient
    assert ((dz.double() - want).abs() <= want.abs() * 32 * torch.finfo(dtype).eps).all()
    size = 0.25 * far / 2.0
    assert ((loss.double() - size).abs() <= size * 4 * torch.finfo(dtype).eps + 3.0).all()


def test_reference_masks():
    z = torch.randn(4, 6, dtype=torch.float64)
    z[0, 1:4] = -math.inf
    z[1] = -math.inf
    z[2] = torch.finfo(torch.float32).min
    lp, ent, tlp, tid = kf.token_logprobs_ref(z, torch.tensor([1, 1, 1, 7]), top_k=5)
    keep = z[0, [0, 4, 5]].softmax(-1)
    assert lp[0] == -math.inf and torch.allclose(ent[0], -(keep * keep.log()).sum())
    assert tid[0, 3:].tolist() == [1, 2] and tlp[0, 3] == -math.inf
    assert lp[1].isnan() and ent[1].isnan()
    assert torch.allclose(ent[2], torch.tensor(math.log(6), dtype=torch.float64)) and tid[2].tolist() == [0, 1, 2, 3, 4]
    assert lp[3].isnan() and ent[3].isfinite()  # token outside the vocabulary


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(device):
    z = torch.randn(3, 40, device=device)
    tok = torch.zeros(3, dtype=torch.int64, device=device)
    ids = torch.zeros(3, 4, dtype=torch.int64, device=device)
    t = torch.zeros(3, 4, device=device)
    for bad in (dict(top_k=-1), dict(top_k=41), dict(temperature=0.0), dict(temperature=math.nan),
                dict(temperature=-1.0), dict(temperature=math.inf)):
        with pytest.raises(ValueError):
            kf.token_logprobs(z, tok, **bad)
    with pytest.raises(ValueError):
        kf.token_logprobs(z.new_zeros(2, 300), tok[:2], top_k=129)
    with pytest.raises(ValueError):
        kf.token_logprobs(z, tok[:2])
    with pytest.raises(ValueError):
        kf.token_logprobs(z, tok.int())
    with pytest.raises(TypeError):
        kf.token_logprobs(z.double(), tok)
    with pytest.raises(ValueError):
        kf.token_logprobs(z[:, :0], tok)
    with pytest.raises(ValueError):
        kf.token_logprobs(z.new_zeros(1, 1).expand(1, (1 << 19) + 1), tok[:1])
    with pytest.raises(ValueError):
        kf.topk_distillation(z, ids, t, reduction="mean")
    with pytest.raises(ValueError):
        kf.topk_distillation(z, ids, t, weight=torch.ones(3, device=device))
    with pytest.raises(ValueError):
        kf.topk_distillation(z, ids, t, weight=torch.ones(2, device=device), reduction="sum")
    with pytest.raises(ValueError):
        kf.topk_distillation(z, ids.int(), t)
    with pytest.raises(ValueError):
        kf.topk_distillation(z, ids, t[:, :3])
    with pytest.raises(ValueError):
        kf.topk_distillation(z, ids, ids)
    with pytest.raises(ValueError):
        kf.topk_distillation(z, ids[:, :0], t[:, :0])
    with pytest.raises(ValueError):
        kf.topk_distillation(z, ids.repeat(1, 40), t.repeat(1, 40))
    with pytest.raises(ValueError):
        kf.topk_distillation(z, ids, t, temperature=0)


def test_native_refusals_without_a_gpu():
    """The native entry points raise Python's errors, numbers in their messages included, before they touch a device."""

    from koochak_b200.ops import available, native

    if not available():
        pytest.skip("native library not built")
    z, tok = torch.randn(3, 40), torch.zeros(3, dtype=torch.int64)
    ids, t = torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, 4)
    with pytest.raises(ValueError, match="temperature .* got 0.0"):
        native().token_logprobs(z, tok, 0, 0.0, IGNORE)
    with pytest.raises(ValueError, match="got 41"):
        native().token_logprobs(z, tok, 41, 1.0, IGNORE)
    with pytest.raises(ValueError, match=r"shape \[3\]"):
        native().token_logprobs(z, tok[:2], 0, 1.0, IGNORE)
    with pytest.raises(TypeError, match="Double"):
        native().token_logprobs(z.double(), tok, 0, 1.0, IGNORE)
    with pytest.raises(ValueError, match=r"\[3\]"):
        native().topk_distillation(z, ids, t, 1.0, False, z[0], True)
    with pytest.raises(RuntimeError, match="CUDA"):
        native().topk_distillation(z, ids, t, 1.0, False, None, False)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_leading_shapes_and_empty_batches(device):
    z = _logits(6, 50, torch.float32, "contiguous", device=device).view(2, 3, 50)
    tok = _tokens(6, 50, device, ignored=False).view(2, 3)
    res = kf.token_logprobs(z, tok, top_k=3)
    assert res.logprobs.shape == (2, 3) and res.top_ids.shape == (2, 3, 3)
    loss = kf.topk_distillation(z, res.top_ids, res.top_logprobs, tail=True)
    assert loss.shape == (2, 3)
    # A student that is its own teacher: 2^-19 covers the roundings of q and p against one another.
    assert loss.abs().max() < 2.0**-19
    one = kf.token_logprobs(z[0, 0], tok[0, 0], top_k=2)
    assert one.logprobs.shape == () and one.top_ids.shape == (2,)
    for empty in (z[:0], z[:, :0]):
        lead = empty.shape[:-1]
        e = kf.token_logprobs(empty, tok.new_zeros(lead), top_k=2)
        assert e.logprobs.shape == lead and e.top_ids.shape == (*lead, 2)
        assert kf.topk_distillation(empty, tok.new_zeros(*lead, 4), z.new_zeros(*lead, 4)).shape == lead
        assert kf.topk_distillation(empty, tok.new_zeros(*lead, 4), z.new_zeros(*lead, 4), reduction="sum") == 0


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("tail", [False, True])
def test_gradients_of_rows_left_out(device, tail):
    """Zeros, whatever the rows hold: an ignored token, no slots, weight zero (whose teacher may be anything too)."""

    z = _logits(4, 300, torch.float32, "contiguous", device=device)
    z[0], z[2] = math.nan, math.inf
    z.requires_grad_()
    tok = torch.tensor([IGNORE, 3, IGNORE, 4], device=device)
    ids, t = _teacher(4, 300, 5, tail, ragged=False, device=device)
    none = ids.masked_fill(torch.tensor([[True], [False], [True], [False]], device=device), -1)
    weight = torch.tensor([0.0, 1.0, 0.0, 0.5], device=device)
    bad = t.clone()
    bad[0] = math.nan
    bad[2] = math.inf
    res = kf.token_logprobs(z, tok, ignore_index=IGNORE)
    for total in (res.logprobs.sum() + res.entropy.sum(), kf.topk_distillation(z, none, bad, tail=tail).sum(),
                  kf.topk_distillation(z, none, bad, tail=tail, reduction="sum"),
                  kf.topk_distillation(z, ids, bad, tail=tail, weight=weight, reduction="sum")):
        (dz,) = torch.autograd.grad(total, z)
        assert total.isfinite() and dz.isfinite().all()
        assert not dz[::2].any() and dz[1::2].any(1).all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [50, 5000, 20000])
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_gradient_without_student_mass_off_the_list(device, dtype, vocab, reduction):
    """With a tail and every token off the list masked, the loss is infinite and the rest adds nothing to the gradient,
    which is (Q p - q) / T. Three numbers of at most 1, each accurate to 2^-18, and half a step of the logits' type."""

    rows, k, temperature = 160, 6, 2.0
    gen = torch.Generator().manual_seed(2)
    ids = torch.stack([torch.randperm(vocab, generator=gen)[:k] for _ in range(8)]).repeat(rows // 8, 1)
    t = torch.log_softmax(torch.randn(8, k + 1, generator=gen), -1)[:, :k].repeat(rows // 8, 1)
    z = torch.full((rows, vocab), -math.inf).scatter_(1, ids, torch.randn(8, k, generator=gen).repeat(rows // 8, 1))
    z = z.to(device, dtype).requires_grad_()
    loss = kf.topk_distillation(z, ids.to(device), t.to(device), temperature=temperature, tail=True,
                                reduction=reduction)
    (dz,) = torch.autograd.grad(loss.sum(), z)
    assert (loss == math.inf).all()
    q = torch.zeros(rows, vocab, dtype=torch.float64).scatter_(1, ids, t.double().exp())
    p = torch.softmax(z.detach().cpu().double() / temperature, 1)
    want = (q.sum(1, keepdim=True) * p - q) / temperature
    _close(dz, want, 2.0**-16 / temperature + want.abs() * _half_step(dtype) * 1.01, "dlogits")


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", [-math.inf, "lowest"])
@pytest.mark.parametrize("vocab,left,k", [(40, 7, 7), (5000, 60, 64), (20000, 100, 128)])
def test_teacher_that_lists_every_token_left(device, dtype, mask, vocab, left, k):
    """Teacher and student under one mask that leaves no more tokens than the teacher has slots. What one minus the sum
    of its probabilities is then is rounding: the loss is that of the tokens left, and so is the gradient. Tolerances as
    in _check_distill, of log probabilities below 24 (logits of about 8 and down to -8); a rest of up to 2^-18 that is
    found or not changes a finite log probability's factor, so that the loss may move by as much again."""

    rows = 160
    low = torch.finfo(dtype).min if mask == "lowest" else mask
    masked = torch.ones(rows, vocab, dtype=torch.bool)
    for i in range(rows):
        masked[i, torch.randperm(vocab, generator=torch.Generator().manual_seed(i))[:left]] = False
    teacher, student = (_logits(rows, vocab, dtype, "contiguous", seed=s, device=device)
                        .masked_fill_(masked.to(device), low) for s in (1, 2))
    got = kf.token_logprobs(teacher, top_k=k, temperature=1.5)
    z = student.requires_grad_()
    q = torch.softmax(teacher.cpu().double() / 1.5, 1)
    logp = torch.log_softmax(z.detach().cpu().double() / 1.5, 1)
    want = torch.where(q > 0, q * (q.clamp_min(1e-300).log() - logp.clamp_min(-1e300)), 0.0).sum(1)
    dwant = (logp.exp() - q) / 1.5 / rows
    for reduction in ("none", "sum"):
        loss = kf.topk_distillation(z, got.top_ids, got.top_logprobs, temperature=1.5, tail=True, reduction=reduction)
        (dz,) = torch.autograd.grad(loss.sum() / rows, z)
        goal = want if reduction == "none" else want.sum()
        _close(loss.detach(), goal, (24 + 16) * 2.0**-18 * (1 if reduction == "none" else rows), "loss")
        tol = 2.0**-16 / rows + dwant.abs() * _half_step(dtype) * 1.01 + torch.finfo(dtype).tiny * _half_step(dtype) * 2
        _close(dz, dwant, tol, "dlogits")


# ------------------------------------------------------- log probabilities


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,layout", [
    (1, 1, "contiguous"), (3, 2, "contiguous"), (2, 7, "offset"), (5, 129, "offset"), (4, 1000, "padded"),
    (7, 1001, "contiguous"), (6, 4099, "offset"), (3, 8193, "columns"), (5, 32000, "padded"), (4, 50257, "contiguous"),
    (300, 4099, "contiguous"), (2, 131072, "padded"), (1, 524288, "padded"),
])
def test_logprobs_shapes(dtype, rows, vocab, layout):
    z = _logits(rows, vocab, dtype, layout)
    _check_logprobs(z, _tokens(rows, vocab), top_k=min(5, vocab))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [128, 1000, 4100, 4500, 50257])
@pytest.mark.parametrize("top_k", [1, 2, 31, 33, 128])
def test_alternatives(dtype, vocab, top_k):
    _check_logprobs(_logits(5, vocab, dtype, "contiguous", seed=top_k), None, top_k=top_k, grads=top_k == 2)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [0.05, 0.7, 3.0, 100.0])
def test_logprobs_temperature(dtype, temperature):
    z = _logits(6, 5000, dtype)
    # Logits up to about 16 / 0.05: the log probabilities grow with 1 / T, and their error with them.
    _check_logprobs(z, _tokens(6, 5000), top_k=7, temperature=temperature)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,layout", [(12, 1003, "offset"), (12, 50257, "padded"), (3, 50257, "contiguous"),
                                               (500, 4099, "contiguous")])
def test_likely_tokens_keep_their_digits(dtype, rows, vocab, layout):
    """-log p and the entropy of a token that has nearly all of the probability, relative to their own size.

    -log p = log(1 + rest / e): the rest is a sum of terms 2^x, off by 2^-22 and by ln 2 |x| 2^-24 with |x| below 64,
    relative, 2^-18 together; as much again for its sum, the ratio and the logarithm. The entropy's terms carry the
    same once more through x. The reference takes the rest apart too: 1 + 1e-10 loses digits in 64 bits already."""

    z = _logits(rows, vocab, dtype, layout, sigma=1.0)
    tok = _tokens(rows, vocab, ignored=False)
    tok[0], tok[1], tok[2] = 0, vocab - 1, min(8, vocab - 1)
    z.scatter_(1, tok[:, None], (torch.arange(rows, device=DEV) % 12 * 2.0 + 12.0)[:, None].to(dtype))
    res = kf.token_logprobs(z, tok)
    d = z.double() - z.double().gather(1, tok[:, None])
    e = d.exp().scatter_(1, tok[:, None], 0.0)
    logp = -torch.log1p(e.sum(1))
    ent = (-logp - (e * d).sum(1) / (1 + e.sum(1))).cpu()
    logp = logp.cpu()
    assert (logp > -0.6).any() and (rows < 12 or (logp > -1e-8).any())
    likely = logp > math.log(0.5) + 1e-3
    _close(res.logprobs.cpu()[likely], logp[likely], logp[likely].abs() * 2.0**-17, "logprobs")
    _close(res.entropy.cpu()[likely], ent[likely], ent[likely] * 2.0**-16, "entropy")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,layout", [(12, 1003, "offset"), (12, 50257, "padded"), (3, 50257, "contiguous"),
                                               (500, 4099, "contiguous"), (400, 17, "offset"), (700, 32001, "contiguous")])
@pytest.mark.parametrize("given", [False, True])
def test_likely_alternatives_and_entropies_keep_their_digits(dtype, rows, vocab, layout, given):
    """The same for the most likely alternative and the entropy where another token is given or none; tolerances as
    above. Nothing has a positive log probability or a negative entropy."""

    z = _logits(rows, vocab, dtype, layout, sigma=1.0)
    likely = _tokens(rows, vocab, ignored=False)
    likely[0], likely[1], likely[2] = 0, vocab - 1, min(8, vocab - 1)
    z.scatter_(1, likely[:, None], (torch.arange(rows, device=DEV) % 12 * 2.0 + 12.0)[:, None].to(dtype))
    tok = (likely + 1) % vocab if given else None
    d = z.double() - z.double().gather(1, likely[:, None])
    e = d.exp().scatter_(1, likely[:, None], 0.0)
    logp = -torch.log1p(e.sum(1))
    ent = -logp - (e * d).sum(1) / (1 + e.sum(1))
    sure = logp > math.log(0.5) + 1e-3
    assert sure.any()
    for top_k in (0, 1, 7):
        res = kf.token_logprobs(z, tok, top_k=top_k)
        _close(res.entropy[sure], ent[sure], (ent[sure] * 2.0**-16).cpu(), "entropy")
        assert (res.entropy >= 0).all() and (not given or (res.logprobs <= 0).all())
        if given:
            want = logp + d.gather(1, tok[:, None])[:, 0]
            _close(res.logprobs, want, _logprob_tol(want.cpu()), "logprobs")
        if top_k:
            assert torch.equal(res.top_ids[sure, 0], likely[sure]) and (res.top_logprobs <= 0).all()
            _close(res.top_logprobs[sure, 0], logp[sure], (logp[sure].abs() * 2.0**-17).cpu(), "top_logprobs")
            same = kf.token_logprobs(z, res.top_ids[:, 0].contiguous())
            # one token's log probability, in either place: within both tolerances of the exact value
            first = res.top_logprobs[:, 0]
            _close(same.logprobs, first, torch.where(first > -0.69, first.abs() * 2.0**-16, 2 * _logprob_tol(first)),
                   "places")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [2, 33, 5000, 50257])
def test_two_tokens_with_all_of_the_probability(dtype, vocab):
    """Equal logits side by side (in one thread's share, most often) and apart: neither has more than half."""

    for first, second in ((0, 1), (vocab // 2, vocab // 2 + 1 if vocab > 2 else 0), (0, vocab - 1)):
        z = torch.full((150, vocab), -math.inf, device=DEV, dtype=dtype)
        z[:, first] = z[:, second] = torch.linspace(-30, 30, 150, device=DEV).to(dtype)
        res = kf.token_logprobs(z, torch.full((150,), second, device=DEV), top_k=2, temperature=0.7)
        for got in (-res.logprobs, res.entropy, -res.top_logprobs[:, 0], -res.top_logprobs[:, 1]):
            _close(got, torch.full((150,), math.log(2.0)), 2.0**-20, "ln 2")
        assert (res.top_ids.sort(1).values == torch.tensor(sorted((first, second)), device=DEV)).all()


def _hard_rows(vocab, dtype, device):
    """Rows where selection and sums can go wrong: ties, masks, order in memory, extremes."""

    low = torch.finfo(dtype).min
    gen = torch.Generator().manual_seed(3)
    r = torch.randn(vocab, generator=gen)
    asc = torch.linspace(-9, 9, vocab)
    rows = [
        torch.zeros(vocab),                                        # every value the same
        asc, asc.flip(0),                                          # sorted in memory
        torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0),      # zeros of both signs are ties
        torch.where(torch.arange(vocab) < vocab - 3, -math.inf, r),    # fewer tokens left than alternatives
        torch.where(torch.arange(vocab) == vocab // 2, 1.0, -math.inf),  # one token left
        torch.full((vocab,), low),                                 # masked by the lowest value throughout
        torch.where(torch.arange(vocab) % 7 == 3, r, low),
        torch.round(r),                                            # few distinct values
        torch.where(torch.arange(vocab) < 150, 5.0 + r, r - 9.0),  # the likely ones side by side
        torch.where(torch.arange(vocab) % 512 == 5, 4.0 + r, r),   # ... or in one thread's share
        torch.where(torch.arange(vocab) % 4096 < 8, 4.0 + r, r),
        r * 1e-3, r.clamp(-1, 1) * 1000,
    ]
    return torch.stack(rows).to(dtype).to(device)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [200, 3001, 40001])
@pytest.mark.parametrize("top_k", [3, 128])
def test_hard_rows(dtype, vocab, top_k):
    z = _hard_rows(vocab, dtype, DEV)
    _check_logprobs(z, _tokens(len(z), vocab, ignored=False), top_k=top_k)


def _far_rows(vocab, dtype):
    """Logits, or masks other than the type's lowest value, so large that a product with 1 / T has no digits below one."""

    big = [v for v in (3e4, 1e7, 2e7, 1e9, 1e10, 1e15, 1e30, 1e37, 3e38) if v < torch.finfo(dtype).max]
    r = torch.randn(vocab, generator=torch.Generator().manual_seed(4))
    at = torch.arange(vocab)
    rows = []
    for v in big:
        rows += [torch.full((vocab,), v), torch.full((vocab,), -v),   # one value throughout
                 torch.where(at < vocab // 2, -v, r),                 # masked in front, behind, and here and there
                 torch.where(at < vocab // 2, r, -v), torch.where(at % 3 == 0, r, -v),
                 torch.where(at == vocab // 3, v, r),                 # one far above
                 (r / 4).clamp(-1, 1) * v, v * (1 + r.clamp(-1, 1) * 2.0**-7).clamp(max=1.0)]
    return torch.stack(rows).to(dtype).to(DEV)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [70, 3001, 40001])
@pytest.mark.parametrize("temperature", [1.0, 0.3])
def test_far_logits_and_masks(dtype, vocab, temperature):
    z = _far_rows(vocab, dtype)
    wide = z.double()
    wide = (wide.amax(1) - wide.amin(1)) / temperature > 3e38  # log probabilities beyond fp32 are infinite
    for top_k in (0, 9):
        got = kf.token_logprobs(z[wide], _tokens(int(wide.sum()), vocab, ignored=False), top_k=top_k,
                                temperature=temperature)
        want = kf.token_logprobs_ref(z[wide].double(), _tokens(int(wide.sum()), vocab, ignored=False), top_k=top_k,
                                     temperature=temperature)
        for a, b in zip(got, (want[0], want[1], want[2], want[3])):
            if a is not None:
                _close(a, b.float(), _logprob_tol(b.float().double()) + 2.0**-16, "beyond fp32")
    z = z[~wide]
    rows = len(z)
    for top_k in (0, 9):
        _check_logprobs(z, _tokens(rows, vocab, ignored=False), top_k=top_k, temperature=temperature, grads=top_k == 0)
    ids, t = _teacher(rows, vocab, 8, False, ragged=False)
    ids[:, 0] = z.float().argmax(1)
    q = torch.log_softmax(torch.randn(rows, 9, generator=torch.Generator().manual_seed(6)), -1)[:, :8].to(DEV)
    # Losses one by one: of all rows together only the largest, 1e30, would be looked at. As in _check_distill, with
    # |log p| up to the loss's own size over the least q (2^-6 or more of these), and 24 where that is less.
    for tail, teacher in ((False, t), (True, q)):
        want = kf.topk_distillation_ref(z.double(), ids, teacher, temperature=temperature, tail=tail)
        got = kf.topk_distillation(z, ids, teacher, temperature=temperature, tail=tail)
        _close(got, want.float(), 2.0**-14 * want.abs().cpu().clamp(max=3e38) + 40 * 2.0**-20, "loss")
        for n in (1, 200 // rows + 1):  # clusters and staged rows
            many, ids_n, t_n = (x.repeat(n, 1) for x in (z, ids, teacher))
            loss, stats, dz = kf.topk_distillation_grad(many, ids_n, t_n, temperature=temperature, tail=tail)
            _close(loss, want.float().repeat(n), (2.0**-14 * want.abs().cpu().clamp(max=3e38) + 40 * 2.0**-20).repeat(n), "loss")
            zr = z.double().requires_grad_()
            finite = want.isfinite() | tail
            dwant = torch.autograd.grad(kf.topk_distillation_ref(zr, ids, teacher, temperature=temperature, tail=tail)
                                        .nan_to_num(posinf=0.0).sum(), zr)[0][finite].repeat(n, 1)
            tol = 2.0**-16 / temperature + dwant.abs().cpu() * _half_step(dtype) * 1.01
            _close(dz[finite.repeat(n)], dwant, tol, "dlogits")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_distribution(dtype):
    """-inf throughout, a NaN or +inf: NaN results, as the definitions give; NaN ranks first."""

    z = _logits(4, 5003, dtype, "contiguous")
    z[0] = -math.inf
    z[1, 4000] = math.nan
    z[2, 17] = math.inf
    res = kf.token_logprobs(z.requires_grad_(), _tokens(4, 5003, ignored=False), top_k=4)
    assert res.logprobs[:3].isnan().all() and res.entropy[:3].isnan().all()
    assert res.logprobs[3].isfinite() and res.entropy[3].isfinite()
    assert res.top_ids[0].tolist() == [0, 1, 2, 3] and res.top_ids[1, 0] == 4000 and res.top_ids[2, 0] == 17
    assert res.top_logprobs[3].isfinite().all()
    (dz,) = torch.autograd.grad(res.logprobs.sum(), z)
    assert dz[:3].isnan().any(1).all() and dz[3].isfinite().all()


@gpu
def test_rows_left_out_are_not_read():
    """Ignored rows and rows of zero gradient give zeros whatever they hold; tokens outside the vocabulary give NaN."""

    z = _logits(4, 999, torch.bfloat16, "contiguous")
    z[0], z[1] = math.nan, math.nan
    z = z.requires_grad_()
    tok = torch.tensor([IGNORE, 5, 999, -3], device=DEV)
    res = kf.token_logprobs(z, tok, top_k=2)
    assert res.logprobs[0] == 0 and res.entropy[0] == 0 and res.top_ids[0].tolist() == [-1, -1]
    assert res.logprobs[2].isnan() and res.logprobs[3].isnan() and res.entropy[2:].isfinite().all()
    (dz,) = torch.autograd.grad(res.logprobs, z, torch.tensor([1.0, 0.0, 1.0, 0.0], device=DEV), retain_graph=True)
    assert not dz[0].any() and not dz[1].any() and dz[2].isnan().all() and not dz[3].any()
    (dz,) = torch.autograd.grad(res.entropy[3], z)
    assert dz[3].isfinite().all() and dz[3].any() and not dz[:3].any()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_gradients_of_tokens_outside_the_vocabulary(device):
    z = _logits(5, 99, torch.float32, "contiguous", device=device).requires_grad_()
    tok = torch.tensor([99, -3, 7, IGNORE, 1 << 40], device=device)
    res = kf.token_logprobs(z, tok)
    assert res.logprobs.isnan().tolist() == [True, True, False, False, True]
    up = torch.tensor([1.0, 0.0, 1.0, 1.0, -2.0], device=device)
    (dz,) = torch.autograd.grad(res.logprobs, z, up, retain_graph=True)
    assert dz[0].isnan().all() and not dz[1].any() and dz[2].isfinite().all() and not dz[3].any() and dz[4].isnan().all()
    (dz,) = torch.autograd.grad(res.entropy.sum(), z)
    assert dz.isfinite().all() and dz[[0, 1, 2, 4]].any(1).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place_gradients(dtype):
    """The low-level backward calls may overwrite the logits; other columns and rows stay as they were."""

    rows, vocab = 37, 1003
    buf = torch.full((rows + 1, 1024), 7.0, device=DEV, dtype=dtype)
    buf[:rows, :vocab] = _logits(rows, vocab, dtype, "contiguous")
    tok = _tokens(rows, vocab)
    for in_place in (lambda z, out: kf.token_logprobs_backward(
            z, tok, *_lp_saved(z, tok), torch.ones(rows, device=DEV), torch.ones(rows, device=DEV),
            ignore_index=IGNORE, out=out), lambda z, out: _kd_backward(z, out)):
        apart = in_place(buf[:rows, :vocab], None)
        b = buf.clone()
        z = b[:rows, :vocab]
        assert in_place(z, z) is z
        assert torch.equal(z, apart)
        assert (b[rows] == 7).all() and (b[:, vocab:] == 7).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab", [(37, 1003), (20, 20001), (400, 20001)])
def test_loss_and_gradient_in_place(dtype, tail, rows, vocab):
    """Short rows, two kernels, and staged rows: over the logits, or over other columns of their buffer; what lies around
    stays as it was."""

    ld = vocab + 11
    buf = torch.full((rows + 1, 2 * ld), 7.0, device=DEV, dtype=dtype)
    buf[:rows, 3:3 + vocab] = _logits(rows, vocab, dtype, "contiguous")
    ids, t = _teacher(rows, vocab, 9, tail)
    weight = torch.rand(rows, device=DEV) + 0.5
    weight[::4] = 0
    apart = kf.topk_distillation_grad(buf[:rows, 3:3 + vocab], ids, t, weight=weight, tail=tail)
    for first in (3, 3 + ld):
        b = buf.clone()
        got = kf.topk_distillation_grad(b[:rows, 3:3 + vocab], ids, t, weight=weight, tail=tail,
                                        out=b[:rows, first:first + vocab])
        assert all(torch.equal(x, y) for x, y in zip(got, apart))
        b[:rows, first:first + vocab] = buf[:rows, first:first + vocab]
        assert torch.equal(b, buf)


@gpu
def test_outputs_that_overlap_are_refused():
    buf = _logits(6, 64, torch.float32, "contiguous")
    z = buf[:, :20]
    tok = _tokens(6, 20, ignored=False)
    stats, entropy = _lp_saved(z, tok)
    g = torch.ones(6, device=DEV)
    beside = kf.token_logprobs_backward(z, tok, stats, entropy, g, None, out=buf[:, 20:40])  # other columns are fine
    assert torch.equal(beside, kf.token_logprobs_backward(z, tok, stats, entropy, g, None))
    for out in (buf[:, 4:24], buf.flatten()[8:8 + 6 * 32].view(6, 32)[:, :20], buf[0, :20].expand(6, 20)):
        with pytest.raises(RuntimeError, match="overlap"):
            kf.token_logprobs_backward(z, tok, stats, entropy, g, None, out=out)


def _lp_saved(z, tok):
    _, entropy, stats, _, _ = kf.token_logprobs_forward(z, tok, ignore_index=IGNORE)
    return stats, entropy


def _kd_backward(z, out):
    ids, t = _teacher(z.shape[0], z.shape[1], 9, tail=True)
    _, stats = kf.topk_distillation_forward(z, ids, t, tail=True)
    return kf.topk_distillation_backward(z, ids, t, stats, tail=True, out=out)


# ------------------------------------------------------------ distillation


def _teacher(rows, vocab, k, tail, seed=0, ragged=True, device=DEV):
    gen = torch.Generator().manual_seed(seed + 11)
    ids = torch.stack([torch.randperm(vocab, generator=gen)[:k] if k <= vocab else
                       torch.randint(0, vocab, (k,), generator=gen) for _ in range(rows)])
    t = torch.randn(rows, k + 1, generator=gen) * 2
    t = torch.log_softmax(t, -1)[:, :k] if tail else t[:, :k]
    if ragged and k > 2:
        ids[:, 1] = -1
        ids[::3, 2] = vocab + 5
    if ragged and rows > 3:
        ids[3] = -1
    return ids.to(device), t.contiguous().to(device)


def _check_distill(z, ids, t, tail, temperature=1.0, weight=None, scale=1.0, seed=0):
    rows, vocab = z.shape
    z = z.detach().requires_grad_()
    zr = z.detach().cpu().double().requires_grad_()
    want = kf.topk_distillation_ref(zr, ids.cpu(), t.cpu(), temperature=temperature, tail=tail)
    gen = torch.Generator().manual_seed(seed + 5)
    if weight is None:
        loss = kf.topk_distillation(z, ids, t, temperature=temperature, tail=tail)
        g = torch.randn(rows, generator=gen)
        (dz,) = torch.autograd.grad(loss, z, g.to(z.device))
        (dr,) = torch.autograd.grad(want, zr, g.double())
        got = loss.detach()
    else:
        g = weight.cpu() * scale
        total = kf.topk_distillation(z, ids, t, temperature=temperature, tail=tail, weight=weight, reduction="sum")
        (dz,) = torch.autograd.grad(total, z, torch.tensor(scale, device=z.device))
        (dr,) = torch.autograd.grad(want, zr, g.double())
        want = torch.where(weight.cpu() == 0, 0.0, want.detach() * weight.cpu().double())
        got, want = total.detach()[None], want.sum()[None]
        wsum = weight.abs().sum().item()
    # The loss is a mean (sum q <= 1 + rounding) of differences of log q and log p, each as exact as a log probability.
    lp = torch.log_softmax(zr.detach() / temperature, -1)
    size = torch.where(lp.isinf(), 0.0, lp).abs().amax(-1).nan_to_num(0.0).max().item() + 16
    tol = size * 2.0**-20 * (1.0 if weight is None else wsum)
    _close(got, want.detach(), tol, "loss")
    # dz = g / T (Q p - q [- q_rest p / p_rest]): three numbers of at most 1, each accurate to 2^-18.
    tol = g.abs().double()[:, None] / temperature * 2.0**-16 + dr.nan_to_num(0.0).abs() * _half_step(z.dtype) * 1.01
    _close(dz, dr, tol + torch.finfo(z.dtype).tiny * _half_step(z.dtype) * 2, "dlogits")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab,k,layout", [
    (1, 1, 1, "contiguous"), (2, 7, 7, "offset"), (5, 129, 3, "offset"), (4, 1000, 128, "padded"),
    (7, 1001, 16, "contiguous"), (6, 4099, 33, "offset"), (3, 8193, 5, "columns"), (5, 32000, 64, "padded"),
    (4, 50257, 128, "contiguous"), (300, 4099, 8, "contiguous"), (1, 131072, 100, "padded"), (1, 524288, 20, "padded"),
])
def test_distillation_shapes(dtype, tail, rows, vocab, k, layout):
    z = _logits(rows, vocab, dtype, layout)
    ids, t = _teacher(rows, vocab, k, tail)
    _check_distill(z, ids, t, tail, temperature=1.0 if tail else 2.0)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab,layout", [(1, 777, "contiguous"), (37, 1001, "offset"), (9, 50257, "padded"),
                                               (333, 5000, "padded"), (3, 131072, "contiguous"),
                                               (333, 1001, "contiguous"), (700, 8223, "offset"), (160, 50257, "padded"),
                                               (200, 3, "contiguous"), (1200, 9000, "contiguous")])
@pytest.mark.parametrize("scale", [1.0, 0.375])
def test_distillation_weighted_sum(dtype, tail, rows, vocab, layout, scale):
    z = _logits(rows, vocab, dtype, layout)
    ids, t = _teacher(rows, vocab, min(12, vocab - 1), tail)
    weight = torch.rand(rows, device=DEV) + 0.1
    weight[rows // 2::4] = 0
    z[rows // 2::4] = math.nan  # rows of weight zero are left out
    zc = z.clone()
    zc[rows // 2::4] = 0
    z0 = z.detach().requires_grad_()
    a = kf.topk_distillation(z0, ids, t, tail=tail, weight=weight, reduction="sum")
    (da,) = torch.autograd.grad(a, z0)
    assert a.isfinite() and da.isfinite().all() and not da[rows // 2::4].any()
    _check_distill(zc, ids, t, tail, weight=weight, scale=scale)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_repeated_and_masked(dtype, tail):
    """The same id twice, every id of the vocabulary, teachers of -inf, student masks on and off the list."""

    vocab, k = 301, 40
    z = _logits(8, vocab, dtype, "offset")
    ids, t = _teacher(8, vocab, k, tail, ragged=False)
    ids[0, 5], ids[0, 7] = ids[0, 1], ids[0, 1]
    ids[1] = 300
    ids[2, 1:] = -1
    t[3, 4:] = -math.inf
    z[4, ids[4, 3:].sort().values[0]] = -math.inf
    z[5].index_fill_(0, torch.arange(vocab, device=DEV)[~torch.isin(torch.arange(vocab, device=DEV), ids[5])],
                     -math.inf)
    off = torch.arange(vocab, device=DEV)[~torch.isin(torch.arange(vocab, device=DEV), ids[6])]
    z[6].index_fill_(0, off[::2], torch.finfo(dtype).min)
    rows = [0, 2, 3, 4, 6] if tail else list(range(8))
    if tail:  # row 5 has no student mass off the list, row 1 lists one token 40 times: infinite or above one
        inf = kf.topk_distillation(z, ids, t, tail=True)
        assert inf[5] == math.inf
    _check_distill(z[rows], ids[rows], t[rows], tail)
    if not tail:
        t[7] = -math.inf
        assert kf.topk_distillation(z, ids, t)[7] == 0
    small = _logits(2, 6, dtype, "contiguous")
    all_ids = torch.arange(6, device=DEV).repeat(2, 1)
    q = torch.log_softmax(torch.randn(2, 6, device=DEV), -1) + 1e-3  # sums to a little over one: no rest
    if tail:
        _check_distill(small, all_ids, q, True)


@gpu
def test_distillation_rows_without_slots_are_not_read():
    z = torch.full((3, 500), math.nan, device=DEV, dtype=torch.float16)
    z[1] = 1.0
    ids = torch.tensor([[-1, 500], [3, -1], [-7, 1 << 40]], device=DEV)
    z = z.requires_grad_()
    for tail in (False, True):
        loss = kf.topk_distillation(z, ids, torch.zeros(3, 2, device=DEV) - 0.5, tail=tail)
        (dz,) = torch.autograd.grad(loss.sum(), z)
        assert loss[0] == 0 and loss[2] == 0 and loss[1] > 0
        assert not dz[0].any() and not dz[2].any() and dz[1].isfinite().all()


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("left_out", [lambda i: i % 2 == 0, lambda i: i % 2 == 1, lambda i: i < 300, lambda i: i > 40,
                                      lambda i: i % 3 != 0, lambda i: (i // 200) % 2 == 0, lambda i: i >= 0])
@pytest.mark.parametrize("how", ["weight", "slots"])
def test_rows_left_out_in_any_order(tail, left_out, how):
    """Loss and gradient together, blocks taking several rows each, with rows left out between them."""

    rows, vocab = 2500, 2100
    z = _logits(1, vocab, torch.bfloat16, "contiguous").repeat(rows, 1)
    z += torch.randn_like(z[:, :1])
    ids, t = _teacher(1, vocab, 7, tail, ragged=False)
    ids, t = ids.repeat(rows, 1), t.repeat(rows, 1)
    out = torch.tensor([left_out(i) for i in range(rows)], device=DEV)
    weight = torch.rand(rows, device=DEV) + 0.5
    if how == "weight":
        weight[out] = 0
    else:
        ids[out] = -1
    loss, stats, dz = kf.topk_distillation_grad(z, ids, t, weight=weight, tail=tail)
    apart, _ = kf.topk_distillation_forward(z, ids, t, weight=weight, tail=tail)
    assert not loss[out].any() and not dz[out].any() and (stats[~out, 7] == 1).all()
    # Both kernels are within the loss's tolerance of the exact value (16 + log V covers |log p| here).
    _close(loss, apart, 2 * weight.double().cpu() * (16 + math.log(vocab)) * 2.0**-20, "loss")
    back = kf.topk_distillation_backward(z, ids, t, stats, row_scale=weight, tail=tail)
    assert torch.equal(back, dz)


def _kernels(f):
    """Names of the CUDA kernels that a call launches (none where the profiler sees none)."""

    f()
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        f()
        torch.cuda.synchronize()
    return {e.key for e in prof.key_averages()}


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype,vocab,ld", [(torch.bfloat16, 17001, 17001), (torch.float16, 33001, 33024),
                                            (torch.float32, 12345, 12345), (torch.bfloat16, 16392, 16397)])
def test_staged_rows_left_out_in_any_order(tail, dtype, vocab, ld):
    """As above, for rows that are staged in shared memory: two blocks per SM take several rows each, and any of a block's
    rows may be left out, by weight, by slots, or by either in turn."""

    rows = 1500
    buf = torch.randn(rows, ld, device=DEV, generator=torch.Generator(DEV).manual_seed(3)).mul_(2).to(dtype)
    z = buf[:, :vocab]
    ids, t = (x.repeat(rows // 10, 1) for x in _teacher(10, vocab, 7, tail, ragged=False))
    base = torch.rand(rows, device=DEV, generator=torch.Generator(DEV).manual_seed(4)) + 0.5
    want_loss, stats = kf.topk_distillation_forward(z, ids, t, tail=tail)
    want = kf.topk_distillation_backward(z, ids, t, stats, row_scale=base, tail=tail)
    names = _kernels(lambda: kf.topk_distillation_grad(z, ids, t, weight=base, tail=tail))
    assert not names or any("distill_grad_kernel" in n for n in names), names
    i = torch.arange(rows, device=DEV)
    for out in (i % 2 == 0, i % 2 == 1, i < 300, i > 40, i % 3 != 0, (i // 200) % 2 == 0, (i // 296) % 2 == 1,
                (i // 296) % 3 != 1, torch.rand(rows, device=DEV) < 0.5, i >= 0, i < 0):
        by_slots = torch.rand(rows, device=DEV) < 0.5
        weight, listed = base.clone(), ids.clone()
        weight[out & ~by_slots] = 0
        listed[out & by_slots] = -1
        x = z.clone()
        x[out] = math.nan  # not read
        loss, kept, dz = kf.topk_distillation_grad(x, listed, t, weight=weight, tail=tail)
        assert not loss[out].any() and not dz[out].any() and not kept[out].any() and (kept[~out, 7] == 1).all()
        # Loss: both kernels within (16 + log V) 2^-20 of the exact value. Gradient: 2^-16 each (see _check_distill), and
        # half a step of the logits' type each, relative.
        _close(loss[~out], (base * want_loss)[~out], 1.5 * (16 + math.log(vocab)) * 2.0**-19, "loss")
        _close(dz[~out], want[~out], 1.5 * 2.0**-15 + 2 * _half_step(dtype) * want[~out].double().abs().cpu(), "dlogits")


def _relative_error_of_p(z, temperature):
    """Bound on the relative error of a probability 2^x / S, x = (z - max) / T / ln 2, per element.

    2^x is off by 2^-22, and by ln 2 |x| (2^-24 three times: the difference, 1 / T, the product). S adds the same of
    its terms, and rounding: a thread (128 or more per row) adds two sums of V / 256 terms, which grow, so the
    additions cost half of that many 2^-24, and some 16 more follow. log2 S is rounded at its own size."""

    v = z.double().nan_to_num(neginf=-1e4) / temperature
    x = (v - v.amax(1, keepdim=True)) / math.log(2.0)
    log2s = torch.logsumexp(v - v.amax(1, keepdim=True), 1, keepdim=True) / math.log(2.0)
    return 2.0**-21 + (3 * x.abs() + 3 * log2s + 16 + z.shape[1] / 512) * 2.0**-24


def _output_tol(want, dtype):
    """Half a step of a normal or subnormal result."""

    return want.abs() * _half_step(dtype) * (1 + 2.0**-10) + torch.finfo(dtype).tiny * _half_step(dtype)


SMALL_P = [(3, 129, "offset"), (5, 32000, "padded"), (4, 50257, "contiguous"), (300, 4099, "contiguous"),
           (400, 9001, "offset"), (700, 20011, "contiguous"), (160, 50257, "padded"), (2, 131072, "padded")]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,layout", SMALL_P)
@pytest.mark.parametrize("which", ["logprobs", "entropy", "both"])
def test_every_element_of_logprob_gradients(dtype, rows, vocab, layout, which):
    """Each element to its own size: most are products with a probability of 1e-6, which a tolerance of the row's largest
    would let pass as zeros. Three factors make up dz = (g hot - p (g + gh (ln p + H))) / T."""

    temperature = 1.25
    z = _logits(rows, vocab, dtype, layout).requires_grad_()
    tok = _tokens(rows, vocab)
    gen = torch.Generator(DEV).manual_seed(8)
    g = torch.randn(rows, device=DEV, generator=gen) * (which != "entropy")
    gh = torch.randn(rows, device=DEV, generator=gen) * (which != "logprobs")
    res = kf.token_logprobs(z, tok, temperature=temperature)
    (dz,) = torch.autograd.grad((res.logprobs, res.entropy), z, (g, gh))
    step = max(1, 2**24 // vocab)
    for i in range(0, rows, step):
        part = slice(i, i + step)
        zp = z.detach()[part].double()
        logp = torch.log_softmax(zp / temperature, 1)
        p, counted = logp.exp(), (tok[part] != IGNORE)[:, None]
        h = -(p * logp).sum(1, keepdim=True)
        a, b = g[part].double()[:, None], gh[part].double()[:, None]
        hot = torch.zeros_like(p).scatter_(1, tok[part].clamp_min(0)[:, None], 1.0)
        want = torch.where(counted, (a * (hot - p) - b * p * (logp + h)) / temperature, 0.0)
        rel = _relative_error_of_p(zp, temperature)
        # p's own error in the product, that of ln p (the same) and of H (as at the top of this file) beside it
        inner = rel + (h + math.log(vocab)) * 2.0**-20 + 2.0**-19 + logp.abs() * 2.0**-22
        tol = p * (rel * (a.abs() + b.abs() * (logp.abs() + h)) + inner * b.abs() + 2.0**-22 * (a.abs() + b.abs() * h))
        tol = (tol + hot * a.abs() * 2.0**-22 + 2.0**-124 * (a.abs() + b.abs() * 100)) / temperature
        _close(dz[part], want, (tol + _output_tol(want, dtype)).cpu(), f"rows {i}")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,layout", SMALL_P)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("how", ["none", "sum", "scaled"])
def test_every_element_of_distillation_gradients(dtype, rows, vocab, layout, tail, how):
    """The same for dz = g / T ((Q + r) p - q - [off the list] r p / p_r): each of the three terms is accurate to its
    probability's relative error, and the teacher's q and rest r to 2^-20 (of one, for the rest)."""

    temperature = 1.0 if tail else 2.0
    z = _logits(rows, vocab, dtype, layout).requires_grad_()
    ids, t = _teacher(rows, vocab, 12, tail)
    weight = torch.rand(rows, device=DEV, generator=torch.Generator(DEV).manual_seed(8)) + 0.5
    if how == "none":
        loss = kf.topk_distillation(z, ids, t, temperature=temperature, tail=tail)
        (dz,) = torch.autograd.grad(loss, z, weight)
    else:
        loss = kf.topk_distillation(z, ids, t, temperature=temperature, tail=tail, weight=weight, reduction="sum")
        factor = 1.0 if how == "sum" else 0.375
        (dz,) = torch.autograd.grad(loss, z, torch.full((), factor, device=DEV))
        weight = weight * factor
    step = max(1, 2**24 // vocab)
    for i in range(0, rows, step):
        part = slice(i, i + step)
        zp = z.detach()[part].double()
        p = torch.softmax(zp / temperature, 1)
        valid = (ids[part] >= 0) & (ids[part] < vocab)
        tp = t[part].double().masked_fill(~valid, -math.inf)
        q = tp.exp() if tail else torch.softmax(tp / temperature, 1).nan_to_num(0.0)
        at = torch.where(valid, ids[part], 0)
        listed = torch.zeros_like(p).scatter_add_(1, at, q)
        off = torch.zeros_like(p).scatter_add_(1, at, valid.double()) == 0
        total = q.sum(1, keepdim=True)
        rest = (1 - total).clamp_min(0.0) if tail else torch.zeros_like(total)
        share = torch.where(off, p, 0.0)
        share = share / share.sum(1, keepdim=True) if tail else torch.zeros_like(p)
        w = torch.where(valid.any(1), weight[part], 0.0).double()[:, None] / temperature
        want = w * ((total + rest) * p - listed - rest * share)
        rel = _relative_error_of_p(zp, temperature) + 2.0**-22
        tol = rel * ((total + rest) * p + 2 * rest * share) + 2.0**-20 * (p + share * bool(tail) + 2 * listed)
        _close(dz[part], want, (w * (tol + 2.0**-124) + _output_tol(want, dtype)).cpu(), f"rows {i}")


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows", [148, 200, 296, 600])
@pytest.mark.parametrize("how", ["weight", "slots"])
def test_blocks_whose_only_rows_are_left_out(tail, rows, how):
    """Staged rows (34 KB) that all are left out, most blocks with a single one: nothing between the fetching warp's first
    two messages takes time there. Many launches, as the order of the warps differs from one to the next."""

    vocab = 17001
    z = torch.full((rows, vocab), math.nan, device=DEV, dtype=torch.bfloat16)
    ids, t = _teacher(rows, vocab, 5, tail, ragged=False)
    weight = torch.ones(rows, device=DEV)
    if how == "weight":
        weight[:] = 0
    else:
        ids[:] = -1
    out = torch.empty_like(z)
    for _ in range(50):
        loss, stats, dz = kf.topk_distillation_grad(z, ids, t, weight=weight, tail=tail, out=out.fill_(1.0))
        assert not loss.any() and not stats.any() and not dz.any()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("vocabs", [(50257, 32000, 50257), (25001, 50257, 20000, 40000, 25001)])
def test_vocabularies_one_after_another(dtype, tail, vocabs):
    """One kernel with more shared memory, less, and more again. Twenty different rows, repeated until blocks of
    different SMs take them; rows at the same 16-byte boundaries (160 odd rows further on) have the same results."""

    if dtype == torch.float32:
        vocabs = [v // 2 for v in vocabs]
    known = {}
    for vocab in vocabs:
        z = _logits(20, vocab, dtype, "padded").repeat(10, 1)
        ids, t = (x.repeat(10, 1) for x in _teacher(20, vocab, 11, tail))
        weight = torch.rand(20, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).add_(0.5).repeat(10)
        _check_distill(z, ids, t, tail, weight=weight)
        got = kf.topk_distillation_grad(z, ids, t, weight=weight, tail=tail)
        assert all(torch.equal(a[:20], a[160:180]) for a in got)
        if vocab in known:
            assert all(torch.equal(a, b) for a, b in zip(got, known[vocab]))
        known[vocab] = got


@gpu
def test_two_host_threads():
    """Two vocabularies in two threads with a stream each, every call setting up the kernels anew for its sizes."""

    import threading

    work = []
    for vocab, tail in ((50257, True), (20001, True), (33001, False), (270000, True)):
        rows = 200 if vocab < 100000 else 400
        z = _logits(20, vocab, torch.bfloat16, "padded").repeat(rows // 20, 1)
        ids, t = (x.repeat(rows // 20, 1) for x in _teacher(20, vocab, 11, tail))
        work.append((z, ids, t, tail))

    def call(z, ids, t, tail):
        x = z.detach().requires_grad_()
        loss = kf.topk_distillation(x, ids, t, tail=tail, reduction="sum")
        return loss.detach(), torch.autograd.grad(loss, x)[0], *kf.token_logprobs(z, ids[:, 0].contiguous(), top_k=7)

    want = [call(*w) for w in work]
    torch.cuda.synchronize()
    errors = []

    def run(first):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(24):
                    n = (first + i) % len(work)
                    got = call(*work[n])
                    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(got, want[n])), n
        except BaseException as e:  # noqa: BLE001 (raised again below)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in (0, 1, 3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors[0]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_vocabularies_one_after_another(dtype):
    """The same for the loss alone, whose marks take 64 KB of shared memory at the widest vocabulary."""

    for vocab in (1 << 19, 300000, 1 << 19, 270000, 400000):
        z = _logits(1, vocab, dtype, "contiguous")
        ids, t = _teacher(1, vocab, 20, True, ragged=False)
        want = kf.topk_distillation_ref(z.double(), ids, t, tail=True)
        got = kf.topk_distillation(z.expand(400, -1), ids.expand(400, -1), t.expand(400, -1), tail=True)
        # as in _check_distill: 16 + log V covers |log p| here
        _close(got, want.expand(400), (16 + math.log(vocab)) * 2.0**-20, "loss")


@gpu
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 32776), (torch.bfloat16, 16392), (torch.float32, 16388)])
def test_rows_that_end_at_a_chunk(tail, dtype, vocab):
    """Staged rows with one 16-byte unit more than whole chunks (2048 units) hold, or none where the row starts off a
    boundary: the last chunk is empty for some of a block's rows and not for others."""

    rows = 1500
    few = _logits(10, vocab, dtype, "contiguous")
    buf = torch.empty(rows, vocab + 5, device=DEV, dtype=dtype)[:, 1:1 + vocab]
    buf.copy_(few.repeat(rows // 10, 1))
    units = 16 // few.element_size()
    first = (buf.data_ptr() // few.element_size() + torch.arange(rows) * (vocab + 5)) % units
    head = -first % units
    assert len(set(((vocab - head) // units).tolist())) == 2
    ids, t = _teacher(10, vocab, 9, tail)
    ids, t = ids.repeat(rows // 10, 1), t.repeat(rows // 10, 1)
    want_loss, stats = kf.topk_distillation_forward(buf, ids, t, tail=tail)
    want = kf.topk_distillation_backward(buf, ids, t, stats, tail=tail)
    for _ in range(5):
        loss, _, dz = kf.topk_distillation_grad(buf, ids, t, tail=tail)
        # Loss: both kernels within (16 + log V) 2^-20 of the exact value. Gradient: 2^-16 each (see _check_distill), and
        # half a step of the logits' type each, relative.
        _close(loss, want_loss, (16 + math.log(vocab)) * 2.0**-19, "loss")
        _close(dz, want, 2.0**-15 + 2 * _half_step(dtype) * want.double().abs().cpu(), "dlogits")


@gpu
@pytest.mark.parametrize("tail", [False, True])
def test_every_element_of_a_large_gradient(tail):
    """Loss and gradient together against the two kernels apart, element by element and several times: chunks of a row
    are replaced by the next row's while the gradient is written.

    A dense element is coef 2^x with coef free of cancellation here (no rest): both sides round the same number, known
    to 2^-18, to bf16, so they differ by at most one step, 2^-7 of the value."""

    rows, vocab, k = 16384, 50257, 64
    gen = torch.Generator(DEV).manual_seed(5)
    z = torch.empty(rows, 50304, device=DEV, dtype=torch.bfloat16).normal_(generator=gen).mul_(2)[:, :vocab]
    ids = (torch.randint(0, vocab, (rows, 1), device=DEV, generator=gen) + 7919 * torch.arange(k, device=DEV)) % vocab
    z.scatter_(1, ids, torch.randn(rows, k, device=DEV, generator=gen).add_(8).bfloat16())
    t = torch.log_softmax(torch.randn(rows, k, device=DEV, generator=gen), -1) + 1e-6
    loss, stats = kf.topk_distillation_forward(z, ids, t, tail=tail)
    want = kf.topk_distillation_backward(z, ids, t, stats, tail=tail).scatter_(1, ids, 0.0)
    for _ in range(6):
        got_loss, _, got = kf.topk_distillation_grad(z, ids, t, tail=tail)
        got.scatter_(1, ids, 0.0)
        off = sum(int(((a.float() - b.float()).abs_() > b.float().abs_() * 2.0**-7).sum())
                  for a, b in zip(got.split(2048), want.split(2048)))
        assert off == 0, f"{off} elements"
        assert (got_loss - loss).abs().max() < (16 + math.log(vocab)) * 2.0**-19


@gpu
def test_student_mass_far_below_fp32():
    """The rest's probability is a sum of its own: exact where one minus the listed mass would be zero."""

    z = torch.full((2, 1000), -60.0, device=DEV)
    z[:, :4] = torch.tensor([1.0, 0.5, 0.0, -0.5])
    ids = torch.arange(4, device=DEV).repeat(2, 1)
    t = torch.log(torch.tensor([0.5, 0.2, 0.15, 0.1], device=DEV)).repeat(2, 1)
    _check_distill(z, ids, t, True)


# ----------------------------------------------------------------- together


@gpu
def test_teacher_to_student_run():
    """Alternatives of a teacher feed a student's loss; gradient descent on the student's logits follows the formula."""

    rows, vocab, k = 64, 5003, 32
    teacher = _logits(rows, vocab, torch.bfloat16, "padded", seed=1)
    tok = _tokens(rows, vocab)
    got = kf.token_logprobs(teacher, tok, top_k=k, ignore_index=IGNORE)
    student = _logits(rows, vocab, torch.float32, "contiguous", seed=2)
    _check_distill(student, got.top_ids, got.top_logprobs, True)
    s = student.requires_grad_()
    loss = kf.topk_distillation(s, got.top_ids, got.top_logprobs, tail=True)
    assert (loss[tok == IGNORE] == 0).all()  # ignored rows came back with empty slots
    (g,) = torch.autograd.grad(loss.sum(), s)
    after = kf.topk_distillation(s.detach() - 1e-2 * g, got.top_ids, got.top_logprobs, tail=True)
    assert (after <= loss).all()


@gpu
def test_expanded_logits_and_empty_batches():
    """One row of logits for many tokens (stride zero), whose gradient is the sum; batches of no rows."""

    row = _logits(1, 3001, torch.float32, "contiguous").requires_grad_()
    tok = _tokens(7, 3001, ignored=False)
    ids, t = _teacher(7, 3001, 5, True)
    z = row.expand(7, -1)
    res = kf.token_logprobs(z, tok)
    a, = torch.autograd.grad(res.logprobs.sum() + res.entropy.sum() + kf.topk_distillation(z, ids, t, tail=True).sum()
                             + kf.topk_distillation(z, ids, t, tail=True, reduction="sum"), row)
    rr = row.detach().cpu().double().requires_grad_()
    lp, ent, _, _ = kf.token_logprobs_ref(rr.expand(7, -1), tok.cpu())
    kd = kf.topk_distillation_ref(rr.expand(7, -1), ids.cpu(), t.cpu(), tail=True)
    (lp.sum() + ent.sum() + 2 * kd.sum()).backward()
    # 28 gradients, each within 2^-16 (see _check_distill) of factors of at most 1 + H
    _close(a, rr.grad, 28 * 2.0**-16 * (1 + math.log(3001)), "sum over the expanded rows")
    for dtype in DTYPES:
        e = torch.empty(0, 3001, device=DEV, dtype=dtype, requires_grad=True)
        none = kf.token_logprobs(e, tok[:0], top_k=3)
        total = none.logprobs.sum() + none.entropy.sum() + kf.topk_distillation(e, ids[:0], t[:0]).sum()
        total = total + kf.topk_distillation(e, ids[:0], t[:0], weight=t[:0, 0], reduction="sum")
        total.backward()
        assert total == 0 and e.grad.shape == e.shape


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_widest_vocabulary_in_a_batch(dtype):
    """Two rows of 524288 repeated: blocks of their own instead of the clusters that take the two alone."""

    two = _logits(2, 1 << 19, dtype, "contiguous")
    ids, t = _teacher(2, 1 << 19, 30, True, ragged=False)
    tok = _tokens(2, 1 << 19, ignored=False)
    n = 200
    z = two.repeat(n, 1)
    want = kf.token_logprobs(two, tok, top_k=128)
    got = kf.token_logprobs(z, tok.repeat(n), top_k=128)
    assert torch.equal(got.top_ids, want.top_ids.repeat(n, 1))
    # both within their tolerance of the exact value
    _close(got.logprobs, want.logprobs.repeat(n), 2 * _logprob_tol(want.logprobs.double()).repeat(n), "logprobs")
    loss = kf.topk_distillation(z, ids.repeat(n, 1), t.repeat(n, 1), tail=True)
    one = kf.topk_distillation(two, ids, t, tail=True)
    _close(loss, one.repeat(n), 2 * (16 + math.log(1 << 19)) * 2.0**-20, "loss")
    _check_distill(two, ids, t, True)


@gpu
def test_broadcast_gradients_and_reuse():
    """Expanded upstream gradients, two losses on one set of logits, and backward twice."""

    z = _logits(20, 3001, torch.float32, "contiguous").requires_grad_()
    tok = _tokens(20, 3001, ignored=False)
    ids, t = _teacher(20, 3001, 6, False)
    res = kf.token_logprobs(z, tok)
    loss = kf.topk_distillation(z, ids, t, weight=torch.ones(20, device=DEV), reduction="sum")
    total = res.logprobs.sum() + 0.5 * res.entropy.mean() + loss
    total.backward(retain_graph=True)
    once = z.grad.clone()
    total.backward()
    # Accumulating equal fp32 gradients twice is a doubling, which is exact.
    assert torch.equal(z.grad, 2 * once)
    zr = z.detach().cpu().double().requires_grad_()
    lp, ent, _, _ = kf.token_logprobs_ref(zr, tok.cpu())
    kd = kf.topk_distillation_ref(zr, ids.cpu(), t.cpu())
    (lp.sum() + 0.5 * ent.mean() + kd.sum()).backward()
    _close(once, zr.grad, 3 * 2.0**-16, "sum of gradients")


@gpu
def test_other_stream_and_graph():
    """Work is enqueued on the caller's stream, and forward with backward can be captured and replayed."""

    z = _logits(33, 4099, torch.bfloat16, "padded")
    tok = _tokens(33, 4099)
    ids, t = _teacher(33, 4099, 10, True)
    w = torch.rand(33, device=DEV)

    def step(x):
        x = x.detach().requires_grad_()
        res = kf.token_logprobs(x, tok, top_k=5)
        a, = torch.autograd.grad(res.logprobs.sum() + res.entropy.sum(), x)
        loss = kf.topk_distillation(x, ids, t, tail=True, weight=w, reduction="sum")
        b, = torch.autograd.grad(loss, x)
        return [res.logprobs.detach(), res.entropy.detach(), res.top_ids, a, loss.detach(), b]

    want = step(z)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(z)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    static = z.clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(static)
        graphs.append((g, out))
    other = _logits(33, 4099, torch.bfloat16, "padded", seed=9)
    for data in (z, other):
        static.copy_(data)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        again = step(static)  # the same rows at the same alignment: sums are cut at 16-byte boundaries
        for _, out in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, again))


@gpu
def test_capture_beside_an_eager_graph_of_the_same_leaf():
    """Eager calls and the capture run on one stream, as in the loop's graph mode: the leaf's accumulation node of a graph
    made on the default stream would make torch refuse the capture, whatever the ops are."""

    z = _logits(20, 1003, torch.bfloat16, "contiguous").requires_grad_()
    ids, t = _teacher(20, 1003, 6, True)

    def loss():
        return kf.topk_distillation(z, ids, t, tail=True, reduction="sum") + kf.token_logprobs(z).entropy.sum()

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        alive = loss()
        want = torch.autograd.grad(loss(), z)[0]
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = torch.autograd.grad(loss(), z)[0]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    with torch.cuda.stream(stream):
        (later,) = torch.autograd.grad(alive, z)
    torch.cuda.synchronize()
    assert torch.equal(later, want)


@gpu
@pytest.mark.parametrize("vocab", [1003, 20001])
@pytest.mark.parametrize("captured_forward", [False, True])
def test_backward_captured_apart_from_its_forward(vocab, captured_forward):
    """A backward pass in a graph of its own: every replay is the gradient for the upstream factor of that replay, and
    what was done to an earlier replay's result does not matter."""

    rows = 200
    z = _logits(rows, vocab, torch.bfloat16, "contiguous").requires_grad_()
    ids, t = _teacher(rows, vocab, 6, True)
    w = torch.rand(rows, device=DEV)
    up = torch.ones((), device=DEV)

    def loss():
        return kf.topk_distillation(z, ids, t, tail=True, weight=w, reduction="sum")

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = {f: torch.autograd.grad(loss(), z, torch.full((), f, device=DEV))[0] for f in (1.0, 3.0)}
        eager = None if captured_forward else loss()
    stream.synchronize()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    if captured_forward:
        with torch.cuda.graph(forward, stream=stream):
            eager = loss()
        forward.replay()
    torch.cuda.synchronize()
    with torch.cuda.graph(backward, stream=stream):
        (out,) = torch.autograd.grad(eager, z, up)
    for f in (1.0, 3.0, 1.0, 1.0):
        up.fill_(f)
        backward.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[f]), f
        out.mul_(0.5)  # as clipping by norm does
        torch.cuda.synchronize()


@gpu
def test_repeatable():
    z = _logits(500, 32000, torch.bfloat16)
    tok = _tokens(500, 32000)
    first = kf.token_logprobs(z, tok, top_k=40)
    for _ in range(3):
        again = kf.token_logprobs(z, tok, top_k=40)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    ids, t = first.top_ids, first.top_logprobs
    one = kf.topk_distillation(z, ids, t, tail=True)
    assert torch.equal(one, kf.topk_distillation(z, ids, t, tail=True))


@gpu
def test_offsets_beyond_32_bits():
    """The last rows of a logits buffer of more than 2^32 bytes and more than 2^31 elements."""

    rows, vocab = 17000, 131072
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 20 GB")
    z = torch.zeros(rows, vocab, device=DEV, dtype=torch.bfloat16)
    z[-3:] = _logits(3, vocab, torch.bfloat16, "contiguous")
    tok = torch.full((rows,), IGNORE, device=DEV)
    tok[-3:] = torch.tensor([5, 70000, 131071], device=DEV)
    res = kf.token_logprobs(z, tok, top_k=9)
    small = kf.token_logprobs(z[-3:].clone(), tok[-3:], top_k=9)
    # Few rows are shared by several blocks, so their sums are added in another order: each of the two results is within
    # its tolerance of the exact value, and they are within twice that of one another. The alternatives are equal.
    assert torch.equal(res.top_ids[-3:], small.top_ids)
    for a, b in ((res.logprobs, small.logprobs), (res.top_logprobs, small.top_logprobs)):
        _close(a[-3:], b, 2 * _logprob_tol(b.double()), "log probabilities")
    tol = 2 * ((small.entropy.double() + math.log(vocab)) * 2.0**-20 + 2.0**-19)
    _close(res.entropy[-3:], small.entropy, tol, "entropy")
    assert not res.logprobs[:-3].any()
    ids, t = res.top_ids, res.top_logprobs
    loss, stats = kf.topk_distillation_forward(z, ids, t, tail=True)
    d = kf.topk_distillation_backward(z, ids, t, stats, tail=True, out=z)
    assert not d[:-3].any() and d[-3:].any(1).all()
    del z, d
    rows, vocab = 46000, 50257  # the same for rows that are staged
    z = torch.zeros(rows, vocab, device=DEV, dtype=torch.bfloat16)
    z[-2:] = _logits(2, vocab, torch.bfloat16, "contiguous")
    ids = torch.full((rows, 8), -1, device=DEV)
    ids[-2:], t = _teacher(2, vocab, 8, False, ragged=False)
    t = t.repeat(rows // 2, 1)
    small = z[-2:].clone()
    loss, _, d = kf.topk_distillation_grad(z, ids, t, out=z)
    lone, _, done = kf.topk_distillation_grad(small, ids[-2:], t[-2:], out=small)
    assert not d[:-2].any() and not loss[:-2].any()
    # as in test_every_element_of_a_large_gradient, and twice the gradient's own tolerance on the list
    _close(d[-2:], done, done.double().abs() * 2.0**-7 + 2.0**-15, "dlogits")
    _close(loss[-2:], lone, (16 + math.log(vocab)) * 2.0**-19, "loss")


@gpu
def test_second_derivatives_are_refused():
    z = _logits(3, 64, torch.float32, "contiguous").requires_grad_()
    ids, t = _teacher(3, 64, 4, False, ragged=False)
    for loss in (kf.token_logprobs(z, _tokens(3, 64, ignored=False)).logprobs.exp().sum(),
                 kf.topk_distillation(z, ids, t).square().sum()):
        (g,) = torch.autograd.grad(loss, z, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate"):
            g.sum().backward()


@gpu
def test_second_derivatives_with_a_constant_upstream_gradient_are_refused():
    """A penalty on the gradient of a plain sum: beside other terms it would be left out without a word."""

    z = _logits(3, 64, torch.float32, "contiguous").requires_grad_()
    ids, t = _teacher(3, 64, 4, False, ragged=False)
    for loss in (kf.token_logprobs(z, _tokens(3, 64, ignored=False)).logprobs.sum(), kf.topk_distillation(z, ids, t).sum(),
                 kf.topk_distillation(z, ids, t, reduction="sum")):
        (g,) = torch.autograd.grad(loss, z, create_graph=True)
        (once,) = torch.autograd.grad(z.square().sum() + (2 * z).sum(), z)  # unrelated terms go on working
        assert g.requires_grad and once.isfinite().all()
        with pytest.raises(RuntimeError, match="differentiate"):
            (z.sum() + g.square().sum()).backward()


def _forward_mode(token_logprobs, topk_distillation, device):
    import torch.autograd.forward_ad as fwad

    z, d = torch.randn(2, 3, 40, device=device).unbind()
    ids, t = torch.tensor([[3, 5]] * 3, device=device), torch.zeros(3, 2, device=device)
    with fwad.dual_level():
        for grad in (False, True):
            dual = fwad.make_dual(z.clone().requires_grad_(grad), d)
            for f in (lambda: token_logprobs(dual), lambda: topk_distillation(dual, ids, t)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f()


@gpu
def test_forward_mode_is_refused():
    _forward_mode(kf.token_logprobs, kf.topk_distillation, DEV)


def test_forward_mode_is_refused_without_a_gpu():
    from koochak_b200.ops import available, native

    if not available():
        pytest.skip("native library not built")
    _forward_mode(lambda z: native().token_logprobs(z, None, 0, 1.0, IGNORE),
                  lambda z, ids, t: native().topk_distillation(z, ids, t, 1.0, False, None, False), "cpu")


@gpu
def test_logits_changed_after_the_forward_pass_are_noticed():
    z = _logits(3, 64, torch.float32, "contiguous").requires_grad_()
    y = z * 1.0
    ids, t = _teacher(3, 64, 4, False, ragged=False)
    for loss in (kf.token_logprobs(y).entropy.sum(), kf.topk_distillation(y, ids, t).sum()):
        y.detach().zero_()
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward(retain_graph=True)


# ------------------------------------------------------------------ models


def _small_models(device):
    from koochak_b200.models import GPT2, Llama

    torch.manual_seed(11)
    return [(GPT2(n_layer=2, n_head=4, n_embd=256, vocab_size=1003, block_size=128).to(device),
             GPT2(n_layer=1, n_head=4, n_embd=256, vocab_size=1003, block_size=128).to(device)),
            (Llama(n_layer=2, n_head=4, dim=256, ffn_dim=384, vocab_size=1000, max_seq_len=128).to(device),
             Llama(n_layer=1, n_head=4, dim=256, ffn_dim=384, vocab_size=1000, max_seq_len=128).to(device))]


@pytest.mark.parametrize("which", [0, 1])
def test_models_teacher_and_student_on_cpu(which):
    teacher, student = _small_models("cpu")[which]
    idx = torch.randint(0, 1000, (2, 16))
    targets = torch.randint(0, 1000, (2, 16))
    targets[0, :4] = IGNORE
    with torch.no_grad():
        got = teacher.token_logprobs(idx, targets, top_k=10)
        p = torch.log_softmax(teacher(idx), -1)
    keep = targets != IGNORE
    # fp32 against fp32 of the same formula in another order
    assert torch.allclose(got.logprobs[keep], p.gather(-1, targets.clamp_min(0)[..., None])[..., 0][keep], atol=1e-5)
    assert torch.allclose(got.entropy[keep], -(p.exp() * p).sum(-1)[keep], atol=1e-5)
    assert (got.top_ids[~keep] == -1).all() and not got.logprobs[~keep].any()
    loss = student.distillation_loss(idx, got.top_ids, got.top_logprobs, tail=True)
    loss.backward()
    z = student(idx).detach()
    rows = kf.topk_distillation_ref(z.reshape(-1, z.shape[-1]).double(), got.top_ids.reshape(-1, 10),
                                    got.top_logprobs.reshape(-1, 10), tail=True)
    assert torch.allclose(loss.detach().double(), rows.sum() / keep.sum(), atol=1e-5)
    assert all(q.grad is not None and q.grad.isfinite().all() for q in student.parameters())


@gpu
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_models_teacher_and_student_native(which, dtype):
    """The run as a user makes it: the teacher's alternatives feed the student's loss, on the native kernels, against
    the fp32 reference path; 16-bit activations are compared as the other model tests do."""

    teacher, student = _small_models(DEV)[which]
    idx = torch.randint(0, 1000, (2, 128), device=DEV)
    targets = torch.randint(0, 1000, (2, 128), device=DEV)
    targets[1, 100:] = IGNORE
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        got = teacher.token_logprobs(idx, targets, top_k=16)
    with torch.no_grad():
        ref = teacher.token_logprobs(idx, targets, top_k=16)
    assert (got.logprobs - ref.logprobs).abs().max() < 2e-2 and (got.entropy - ref.entropy).abs().max() < 2e-2

    def grads(native):
        student.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=dtype, enabled=native):
            loss = student.distillation_loss(idx, ref.top_ids, ref.top_logprobs, tail=True)
            lp = student.token_logprobs(idx, targets)
            total = loss - 0.1 * lp.logprobs.mean() - 0.01 * lp.entropy.mean()
        total.backward()
        return loss.item(), {n: q.grad.detach().clone() for n, q in student.named_parameters()}

    loss_n, g_n = grads(True)
    loss_r, g_r = grads(False)
    assert abs(loss_n - loss_r) < 2e-2
    for n in g_r:
        err = ((g_n[n] - g_r[n]).abs().max() / (g_r[n].abs().max() + 1e-6)).item()
        assert err < 0.08, (n, err)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_models_logits_masked_in_place(which, device):
    """Tokens that may not be produced are masked in the logits themselves, and take no gradient."""

    model = _small_models(device)[which][1]
    idx = torch.randint(0, 1000, (2, 64), device=device)
    tok = torch.randint(100, 1000, (2, 64), device=device)

    def step(native):
        model.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=native):
            z = model.logits(idx)
            z[..., :100] = -math.inf
            z[0, :, 700:] += 1.0
            res = kf.token_logprobs(z, tok, top_k=5)
        assert (res.top_ids >= 100).all()
        (-res.logprobs.mean()).backward()
        return res.logprobs.detach(), {n: q.grad.clone() for n, q in model.named_parameters()}

    lp, g = step(device == "cuda")
    lp_r, g_r = step(False)
    assert (lp - lp_r).abs().max() < 2e-2
    for n in g_r:  # as in the test above
        assert ((g[n] - g_r[n]).abs().max() / (g_r[n].abs().max() + 1e-6)).item() < 0.08, n


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_models_logits_with_gradients_of_any_strides(which, device):
    """Upstream gradients that are expanded rows, one number, transposed, or views at odd places."""

    model = _small_models(device)[which][1]
    idx = torch.randint(0, 1000, (2, 64), device=device)
    V = model.config.vocab_size
    rows = torch.randn(1, 1, V, device=device)
    many = torch.randn(64, 2, V, device=device)
    odd = torch.randn(2, 64, V + 9, device=device)
    for g in (rows.expand(2, 64, V), rows[..., :1].expand(2, 64, V), many.transpose(0, 1), odd[..., 3:V + 3],
              many[:1, :1].transpose(0, 1).expand(2, 64, V)):
        got = []
        for native in (device == "cuda", False):
            with torch.autocast("cuda", dtype=torch.bfloat16, enabled=native):
                z = model.logits(idx)
            up = g.to(z.dtype) if g.stride(-1) else g[..., :1].to(z.dtype).expand(2, 64, V)
            if g.stride(1) == 0:
                up = up[:1, :1].expand(2, 64, V)  # a cast of an expanded tensor is expanded no more
            got.append(torch.autograd.grad(z, list(model.parameters()), up))
        for a, b in zip(*got):  # as in the tests above
            assert ((a - b).abs().max() / (b.abs().max() + 1e-6)).item() < 0.08


@gpu
@pytest.mark.parametrize("which", [0, 1])
def test_distillation_through_a_captured_training_step(which):
    """The training loop's captured step: a teacher's alternatives, the student's loss and a policy term, scaled as a loop
    with several micro-steps does. Each replay against an eager step on the same batch and weights, as in the graph
    mode's own test."""

    from koochak_b200.runtime.graphed_step import GraphedStep

    teacher, student = _small_models(DEV)[which]
    gen = torch.Generator().manual_seed(2)
    named = list(student.named_parameters())
    step = GraphedStep(student, warmup=1)

    def batch():
        idx = torch.randint(0, 1000, (4, 65), generator=gen).to(DEV)
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
            got = teacher.token_logprobs(idx[:, :-1].contiguous(), top_k=16)
        return {"idx": idx[:, :-1].contiguous(), "targets": idx[:, 1:].contiguous(), "ids": got.top_ids,
                "logprobs": got.top_logprobs}

    def forward(b):
        kd = student.distillation_loss(b["idx"], b["ids"], b["logprobs"], tail=True)
        lp = student(b["idx"], method="token_logprobs", tokens=b["targets"])
        loss = 0.5 * kd - 0.1 * lp.logprobs.mean() - 0.01 * lp.entropy.mean()
        return {"loss": loss}, loss, loss / 4 * 64

    def eager(b):
        student.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16), step.on_side_stream():
            _, loss, scaled = forward(b)
            scaled.backward()
        return loss.item(), {n: q.grad.detach().clone() for n, q in named}

    def rel(a, b):
        return float((a - b).norm() / (b.norm() + 1e-12))

    eager(batch())
    step.note_eager()
    for i in range(4):
        b = batch()
        want_loss, want = eager(b)
        _, again = eager(b)
        student.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16), step.on_side_stream():
            _, loss = step.run(b, forward)
        assert abs(loss.item() - want_loss) <= 2e-3 * max(1.0, abs(want_loss))
        for n, q in named:
            a, w, r = q.grad.detach(), want[n], again[n]
            if n.endswith("attn.c_attn.bias"):  # the key third's exact gradient is zero
                third = len(a) // 3
                a, w, r = (torch.cat([x[:third], x[2 * third:]]) for x in (a, w, r))
            assert rel(a, w) < max(2e-2, 4 * rel(r, w)), (i, n)
        with torch.no_grad():
            for _, q in named:
                q.mul_(0.99).add_(torch.randn_like(q), alpha=1e-3)
    assert step.graph is not None and not step.disabled
