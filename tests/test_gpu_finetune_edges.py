"""The ends of what the operators of decoder fine-tuning accept: row counts at the edge of 32 bits, exponents beyond fp32, rows at far levels, forms chosen by size, outputs that are inputs.

Tolerances count roundings, as in test_gpu_finetune_ops.py: U = 2^-24 is half a step of fp32, a sum along a tree whose longest path has k additions is off by k U sum|terms| at most."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from novic_amd import ops

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
