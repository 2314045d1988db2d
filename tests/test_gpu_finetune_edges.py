"""The ends of what the operators of decoder fine-tuning accept: row counts at the edge of 32 bits, exponents beyond fp32, rows at far levels, forms chosen by size, outputs that are inputs.

Tolerances count roundings, as in test_gpu_finetune_ops.py: U = 2^-24 is half a step of fp32, a sum along a tree whose longest path has k additions is off by k U sum|terms| at most."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from novic_amd import ops
import test_gpu_finetune_ops as whole  # (its tests at other sizes; imported by name they would be collected here once more)
from test_gpu_finetune_ops import far_rows, half_step, near

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda"
MOST = (1 << 31) - 1  # rows


def pieces(n, size=1 << 28):
	return [slice(a, min(a + size, n)) for a in range(0, n, size)]


def test_layernorm_forward_of_the_most_rows():
	"""2^31 - 1 rows of one bf16 column: the row behind a team's last is no int.  Variance 0: the output is beta, the mean the element itself."""
	x = torch.empty(MOST, 1, dtype=BF16, device=DEV)
	for s in pieces(MOST):
		x[s, 0] = (torch.arange(s.start, s.stop, device=DEV, dtype=torch.int32) % 251).to(BF16)  # exact in bf16
	y, mean, rstd = torch.zeros_like(x), torch.full((MOST,), -1.0, device=DEV), torch.full((MOST,), -1.0, device=DEV)
	ops.layernorm_stats_fwd(x, torch.full((1,), 2.0, device=DEV), torch.full((1,), 0.5, device=DEV), y, mean, rstd, eps=0.25)
	for s in pieces(MOST):
		assert bool((y[s] == 0.5).all()) and bool((mean[s] == x[s, 0]).all()) and bool(((rstd[s] - 2.0).abs() <= 4 * U).all()), s


def test_layernorm_backward_of_the_most_rows():
	"""The same count backward, with mean 0 and rstd 1 given: dx = (g - g) - x (g x) over a row of one column, g = dy.  Small whole numbers, so that every sum is exact; dy is zero
	but for the last rows."""
	x = torch.empty(MOST, 1, dtype=BF16, device=DEV)
	for s in pieces(MOST):
		x[s, 0] = (torch.arange(s.start, s.stop, device=DEV, dtype=torch.int32) % 3 - 1).to(BF16)
	dy = torch.zeros_like(x)
	last = torch.arange(40_000, device=DEV) % 5 - 2
	dy[-40_000:, 0] = last.to(BF16)
	dx = torch.full_like(x, 7.0)
	one, dgamma, dbeta = torch.ones(1, device=DEV), torch.empty(1, device=DEV), torch.empty(1, device=DEV)
	ops.layernorm_stats_bwd(dy, x, one, torch.zeros(MOST, device=DEV), torch.ones(MOST, device=DEV), dx, dgamma, dbeta)
	for s in pieces(MOST):
		assert bool((dx[s] == -x[s] * x[s] * dy[s]).all()), s
	assert float(dgamma) == float((last * x[-40_000:, 0].long()).sum()) and float(dbeta) == float(last.sum())


def test_policy_of_the_most_sequences():
	"""2^31 - 1 sequences of one position, one logit: a sequence's count is taken in steps that end beyond 2^31.  The log-probability is 0; ratio 1, advantages only at the end."""
	logits, target = torch.zeros(MOST, 1, dtype=BF16, device=DEV), torch.zeros(MOST, 1, dtype=torch.int32, device=DEV)
	target[1::2] = -1  # every other position does not count
	old, adv, stats = torch.zeros(MOST, 1, device=DEV), torch.zeros(MOST, device=DEV), torch.empty(4, device=DEV)
	adv[-1000:] = -3.0
	count = (MOST + 1) // 2
	for per_seq in (False, True):
		ops.policy_loss(logits, target, old, adv, stats.fill_(7), per_sequence=per_seq)
		want = 3.0 * 500 / count
		assert abs(float(stats[0]) - want) <= 8 * U * want and float(stats[1]) == 0 and float(stats[2]) == 0 and float(stats[3]) == float(torch.tensor(float(count)))


@pytest.mark.parametrize("per_seq", [False, True])
@pytest.mark.parametrize("V,dtype", [(5, F32), (100, BF16), (1500, F16), (1500, F32), (5000, BF16), (40_000, F32), (70_001, BF16)])
def test_policy_of_large_differences(V, dtype, per_seq):
	"""Ratios and KL terms beyond fp32 (88.7) and beyond fp64 (709) are finite gradients where what they are multiplied with is zero or small: advantages of 0, a KL coefficient
	of 0 (the KL is watched, not trained on), small coefficients; against the definition in 64 bits, where a zero factor leaves the term out."""
	g = torch.Generator(device=DEV).manual_seed(V)
	x = (2.0 * torch.randn(8, V, generator=g, device=DEV)).to(dtype)
	target = torch.randint(0, V, (4, 2), generator=g, device=DEV)
	lse = torch.logsumexp(x.double(), 1)
	lp = (x.double().gather(1, target.view(-1, 1)).squeeze(1) - lse).view(4, 2)
	p = (x.double() - lse[:, None]).exp()
	onehot = torch.zeros_like(p).scatter_(1, target.view(-1, 1), 1.0)
	d_old = torch.tensor([[100.0, 1000.0], [60.0, -100.0], [95.0, 0.1], [-0.5, 0.5]], device=DEV, dtype=torch.double)
	d_ref = torch.tensor([[100.0, -100.0], [1000.0, 0.3], [95.0, -1000.0], [2.0, 0.0]], device=DEV, dtype=torch.double)
	old, ref = (lp - d_old).float(), (lp + d_ref).float()
	adv = torch.tensor([[0.0, 0.0], [-1e-10, 2.0], [-1e-20, 1.0], [-1.0, -0.0]], device=DEV)
	share = torch.full((4, 2), 1 / 8, device=DEV, dtype=torch.double)  # (all positions count: both means are the same)
	for kl in (0.0, 1e-30):
		rr = torch.where(ref - lp > 700, lp + 90.0, ref.double()).float() if kl else ref
		stats, d, out = torch.empty(4, device=DEV), torch.empty_like(x), torch.empty(4, 2, device=DEV)
		ops.policy_loss(x, target, old, adv, stats, clip=(0.2, 0.3), ref=rr, kl_coef=kl, per_sequence=per_seq, dlogits=d, logp=out)
		q, dd, a = (lp - old.double()).exp(), rr.double() - lp, adv.double()
		cut = ((a > 0) & (q > 1.3)) | ((a < 0) & (q < 0.8))
		zero = torch.zeros((), device=DEV, dtype=torch.double)
		gain = torch.where(a == 0, zero, torch.where(cut, torch.where(a > 0, 1.3, 0.8), q) * a)
		term = torch.expm1(dd) - dd
		coef = torch.where(cut, zero, -torch.where(a == 0, zero, q * a)) - (kl * torch.expm1(dd) if kl else zero)
		each = -gain + (kl * term if kl else zero)
		want = (coef * share).view(-1, 1) * (onehot - p)
		# a log-probability is off by (96 + 20) U at most (96 additions, its exponents' distances), its ratio and exp(d) by that much relative, so that the slope expm1(d) of the KL
		# term is off by exp(d) times that; 32 U for all other roundings
		off = 150 * U
		bound = ((coef.abs() + (kl * dd.exp() if kl else zero)) * share).view(-1, 1) * off * (onehot + p) * 2 + want.abs() * (torch.finfo(dtype).eps / 2 + 8 * U) + torch.finfo(dtype).smallest_normal
		held = want.abs() <= torch.finfo(dtype).max  # (infinite where fp16 does not hold it)
		assert torch.isfinite(d[held]).all() and not d.isnan().any()
		assert bool(((d.double() - want).abs() <= bound)[held].all()), (kl, float(((d.double() - want).abs() - bound)[held].max()))
		loss = float((each * share).sum())
		assert math.isfinite(float(stats[0])) and abs(float(stats[0]) - loss) <= off * float((each.abs() * share).sum())
		assert float(stats[2]) == float((cut * share).sum()) and float(stats[3]) == 8
		mean = float((term * share).sum())  # (infinite where fp32 does not hold it)
		assert math.isinf(float(stats[1])) if mean > 3.4028236e38 else abs(float(stats[1]) - mean) <= off * float(((term.abs() + dd.abs()) * share).sum())


def test_policy_of_an_excluded_target():
	"""A target whose logit is -inf: log-probability -inf, ratio 0.  With a KL coefficient of 0 (or no reference) the row's gradient is that of the ratio, a zero, and the loss is finite."""
	x = torch.zeros(2, 300, device=DEV)
	x[0, 7] = float("-inf")
	target, old, adv = torch.tensor([[7, 7]], device=DEV), torch.full((1, 2), -6.0, device=DEV), torch.full((1,), -1.5, device=DEV)
	for ref in (None, torch.full((1, 2), -6.0, device=DEV)):
		stats, d = torch.empty(4, device=DEV), torch.full_like(x, 7.0)
		ops.policy_loss(x, target, old, adv, stats, ref=ref, dlogits=d)
		assert not d[0].any() and torch.isfinite(d).all() and bool(d[1, 7] != 0)
		q = math.exp(6.0) / 300  # the second row's ratio, 1.34: above the range, but the advantage is negative; the first row's is 0 and held at 0.8
		assert abs(float(stats[0]) - (q + 0.8) * 1.5 / 2) <= 1e-5 and float(stats[2]) == 0.5


VOCABULARIES = [5, 130, 500, 900, 1500, 5000, 10007, 20001, 40_001, 70_001]  # every form of the gradient


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", VOCABULARIES)
def test_log_probability_gradient_of_far_rows(V, dtype):
	"""Rows near any level, masked throughout among them: the gradient is that of the row, whose normaliser the fp32 log-sum-exp beside it no longer holds."""
	A, T = 8, 14
	x, target, p, lp, bound = far_rows(A * T, V, dtype)
	target = target.view(A, T)
	g = torch.Generator(device=DEV).manual_seed(V)
	out, lse, d, grad = torch.empty(A, T, device=DEV), torch.empty(A * T, device=DEV), torch.empty_like(x), torch.randn(A, T, generator=g, device=DEV)
	ops.token_logprobs(x, target, out, lse=lse)
	onehot = torch.zeros_like(p).scatter_(1, target.view(-1, 1), 1.0)
	ops.token_logprobs_bwd(x, target, lse, grad, d)
	ref = grad.double().view(-1, 1) * (onehot - p)
	near(d, ref, grad.double().abs().view(-1, 1) * bound[:, None] * (p + onehot) * 3 + half_step(ref, dtype), f"V = {V}")
	ops.token_logprobs_bwd(x, target, lse, grad, x)
	assert torch.equal(x, d)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", VOCABULARIES)
def test_log_probability_gradient_of_offset_rows(V, dtype):
	"""Ordinary logits on levels up to 60 000, where the log-sum-exp's rounding is up to 2^-9 of every probability: the sums' own accuracy, exponents d from the maximum being off by
	d U and a sum by 96 U.  And a log-sum-exp that is not the row's (of a vocabulary of which these are some columns): the gradient takes it as it is, rounding and all."""
	A, T = 5, 16
	g = torch.Generator(device=DEV).manual_seed(V + 1)
	level = torch.tensor([0.0, 200.0, -200.0, 260.0, -300.0, 4000.0, -4000.0, 60_000.0], device=DEV)[torch.arange(A * T, device=DEV) % 8]
	x = (2 * torch.randn(A * T, V, generator=g, device=DEV) + level[:, None]).to(dtype)
	target, grad = torch.randint(0, V, (A, T), generator=g, device=DEV), torch.randn(A, T, generator=g, device=DEV)
	out, lse, d = torch.empty(A, T, device=DEV), torch.empty(A * T, device=DEV), torch.empty_like(x)
	ops.token_logprobs(x, target, out, lse=lse)
	exact = torch.logsumexp(x.double(), 1)
	onehot = torch.zeros(A * T, V, device=DEV, dtype=torch.double).scatter_(1, target.view(-1, 1), 1.0)
	dist = (x.double() - x.double().amax(1, keepdim=True)).abs()
	coef = grad.double().view(-1, 1)
	other = lse + 8.0
	for given, norm, taken in ((lse, torch.where(lse.abs() > 256, exact, lse.double()), lse.abs() <= 256), (other, other.double(), torch.ones_like(lse, dtype=torch.bool))):
		ops.token_logprobs_bwd(x, target, given, grad, d)
		p = (x.double() - norm[:, None]).exp()
		ref = coef * (onehot - p)
		rel = (96 + 12) * U + 2 * U * dist + 3 * U * (given.double().abs() * taken)[:, None]  # (what is taken as given rounds in x - lse)
		bound = coef.abs() * (p * rel + 3 * U * onehot)
		near(d, ref, bound + half_step(ref.abs() + bound, dtype), f"V = {V}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("A,V", [(3, 5), (3, 100), (3, 1500), (3, 5000), (4200, 5000), (3, 70_001)])
def test_log_sum_exp_of_rows_of_nothing(A, V, dtype):
	"""A row of -inf throughout has no probabilities (NaN) and the log-sum-exp -inf, by every form; its neighbours are untouched."""
	x = torch.zeros(A, V, device=DEV, dtype=dtype)
	x[1] = float("-inf")
	out, lse = torch.empty(A, 1, device=DEV), torch.empty(A, device=DEV)
	ops.token_logprobs(x, torch.zeros(A, 1, dtype=torch.int64, device=DEV), out, lse=lse)
	rest = torch.arange(A, device=DEV) != 1
	assert float(lse[1]) == float("-inf") and bool(out[1].isnan().all())
	assert bool(((lse[rest] - math.log(V)).abs() <= 8 * U * math.log(V)).all()) and bool(((out[rest] + math.log(V)).abs() <= 8 * U * math.log(V)).all())


@pytest.mark.parametrize("n,V", [(2, 300), (520, 700), (3, 70_001)])
def test_preference_with_an_excluded_target(n, V):
	"""A rejected label with a token whose logit is -inf: margin +inf, loss and slope 0 without smoothing, an infinite loss with it; for the preferred label the other way round."""
	x = torch.zeros(2 * n, V, device=DEV)
	target, ref = torch.full((2 * n, 1), 3, device=DEV), torch.full((2 * n, 1), -math.log(V), device=DEV)
	x[n, 3] = float("-inf")  # the first pair's rejected label
	stats, margin, d = torch.empty(3, device=DEV), torch.empty(n, device=DEV), torch.full_like(x, 7.0)
	ops.preference_loss(x, target, ref, stats, beta=0.5, margin=margin, dlogits=d)
	assert float(margin[0]) == float("inf") and bool((margin[1:].abs() <= 64 * U * math.log(V)).all())
	want = (n - 1) * math.log(2) / n
	assert abs(float(stats[0]) - want) <= 64 * U * math.log(V) + 8 * U * want and float(stats[1]) == float("inf")
	assert not d[0].any() and not d[n].any() and torch.isfinite(d).all() and bool((d[1:n, 3] < 0).all())
	ops.preference_loss(x, target, ref, stats, beta=0.5, smoothing=0.1)
	assert float(stats[0]) == float("inf")
	x[n, 3], x[0, 3] = 0.0, float("-inf")
	ops.preference_loss(x, target, ref, stats, beta=0.5, margin=margin)
	assert float(margin[0]) == -float("inf") and float(stats[0]) == float("inf")


@pytest.mark.parametrize("n,V", [(2, 300), (520, 700), (3, 70_001)])
def test_preference_of_a_small_beta(n, V):
	"""The square form at beta = 3e-20: loss (1 / (2 beta))^2 = 2.8e38, slope 1 / beta = 3.3e19, both fp32 numbers; their way there (1 / beta^2 = 1.1e39) is not."""
	beta = 3e-20
	x, target, ref = torch.zeros(2 * n, V, device=DEV), torch.full((2 * n, 1), 3, device=DEV), torch.full((2 * n, 1), -math.log(V), device=DEV)
	stats, d = torch.empty(3, device=DEV), torch.empty_like(x)
	ops.preference_loss(x, target, ref, stats, beta=beta, kind="square", dlogits=d)
	assert abs(float(stats[0]) - 0.25 / beta ** 2) <= 8 * U * 0.25 / beta ** 2  # (u, some 1e-6, adds nothing to 1 / (2 beta))
	want = torch.full((2 * n, V), 1.0 / V, device=DEV, dtype=torch.double)
	want[:, 3] -= 1
	want[n:] *= -1
	want *= 1 / beta / n
	near(d, want, (96 + 16) * U * want.abs())


@pytest.mark.parametrize("per_seq", [False, True])
@pytest.mark.parametrize("A,T,V,dtype", [(1300, 7, 97, BF16), (20_000, 5, 33, F32), (20_000, 5, 33, F16), (90, 300, 40, F32), (2500, 40, 65, BF16), (700, 12, 3000, BF16)])
def test_policy_of_many_rows(A, T, V, dtype, per_seq):
	"""Row counts at which the counts come from a launch of their own (several lanes a sequence, several sequences a lane) and the four means from slices."""
	whole.test_policy(A, T, V, 3, 1, dtype, 0.1, 2, per_seq)
	whole.test_policy(A, T, V, 0, 0, dtype, 0.0, 1, per_seq)


@pytest.mark.parametrize("dtype,n,T,V", [(BF16, 4097, 2, 600), (F32, 4099, 3, 300), (F16, 8191, 1, 2500), (BF16, 4097, 9, 700), (F32, 5001, 2, 40)])
def test_preference_of_many_weighted_pairs(dtype, n, T, V):
	"""More pairs than whose weights every workgroup adds up for itself (odd counts: with weights, the first of them 0)."""
	whole.test_preference(n, T, V, 3, 1, dtype, "sigmoid", 0.1, 0.3)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("E", [5, 97, 509, 1280, 5001, 9000, 16384])
def test_layernorm_backward_over_its_inputs(E, dtype):
	"""dx written over x, and over dy, with and without the residual's gradient: the bits of the one written beside them; both affine gradients too."""
	g = torch.Generator(device=DEV).manual_seed(E)
	rows = 700
	rnd = lambda: torch.randn(rows, E, generator=g, device=DEV).to(dtype)  # noqa: E731
	x, dy, resid, gamma = rnd(), rnd(), rnd(), torch.randn(E, generator=g, device=DEV)
	mean, rstd = x.float().mean(1), (x.float().var(1, unbiased=False) + 1e-5).rsqrt()
	for dx_in in (None, resid):
		dx, dgamma, dbeta = torch.empty_like(x), torch.empty(E, device=DEV), torch.empty(E, device=DEV)
		ops.layernorm_stats_bwd(dy, x, gamma, mean, rstd, dx, dgamma, dbeta, dx_in=dx_in)
		for over in ("x", "dy"):
			a, b, dg, db = x.clone(), dy.clone(), torch.empty(E, device=DEV), torch.empty(E, device=DEV)
			out = a if over == "x" else b
			ops.layernorm_stats_bwd(b, a, gamma, mean, rstd, out, dg, db, dx_in=dx_in)
			assert torch.equal(out, dx) and torch.equal(dg, dgamma) and torch.equal(db, dbeta), over
