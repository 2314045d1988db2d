"""The operators of decoder fine-tuning against their definitions in 64 bits: LayerNorm with kept statistics, counter-based dropout, token log-probabilities, the preference and the
policy loss (novic_amd/ops.py), each at the widths, types, strides and masks where it can go wrong, and all together as a fine-tuning step runs them.

Tolerances count roundings.  u = 2^-24 is half a step of fp32; an output of type t adds half a step of t, eps_t / 2 relative (and half the smallest subnormal).  A sum of n fp32 terms
taken along a tree whose longest path has k additions is off by at most k u sum|terms|; the kernels' longest paths are 64 terms in a lane, 6 steps in a wave and 16 waves: K = 96."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from novic_amd import _lib, ops

pytestmark = pytest.mark.gpu
U, K = 2.0 ** -24, 96
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = {"f32": F32, "bf16": BF16, "f16": F16}
DEV = "cuda"


def half_step(ref, dtype):
	"""What rounding to dtype may change."""
	f = torch.finfo(dtype)
	return ref.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def near(got, ref, bound, what=""):
	"""|got - ref| <= bound elementwise; NaN and infinities where ref has them."""
	got = got.double()
	assert got.shape == ref.shape
	odd = ~torch.isfinite(ref)
	assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
	assert torch.equal(got[odd & ~torch.isnan(ref)], ref[odd & ~torch.isnan(ref)]), f"{what}: infinities in other places"
	off = (got - ref).abs()[~odd] - (bound.expand_as(ref) if isinstance(bound, torch.Tensor) else torch.full_like(ref, bound))[~odd]
	assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max()):.3e} over its bound"


class Box:
	"""A matrix inside a larger buffer of sentinels: row padding `extra`, first element `shift` elements behind the buffer's start, rows behind the last."""

	def __init__(self, rows, cols, dtype, extra=0, shift=0, fill=None):
		self.ld = cols + extra
		self.buf = torch.full((shift + (rows + 2) * self.ld,), 77.0, dtype=dtype, device=DEV)
		self.t = self.buf[shift:shift + rows * self.ld].view(rows, self.ld)[:, :cols]
		if fill is not None:
			self.t.copy_(fill)
		self.inside = torch.zeros_like(self.buf, dtype=torch.bool)
		self.inside[shift:shift + rows * self.ld].view(rows, self.ld)[:, :cols] = True

	def intact(self):
		return bool((self.buf[~self.inside] == 77.0).all())


def gen(seed):
	return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=F32, scale=1.0, shift=0.0):
	return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dtype)


# ---- LayerNorm -----------------------------------------------------------------------------------------------------------------------------------------------------

def ln_forward_ref(x, gamma, beta, eps):
	x = x.double()
	mu = x.mean(1, keepdim=True)
	rstd = ((x - mu).square().mean(1, keepdim=True) + eps).rsqrt()
	y = (x - mu) * rstd * gamma.double()
	return (y + beta.double() if beta is not None else y), mu, rstd


def ln_forward_bound(x, gamma, beta, ref, mu, rstd, dtype):
	"""mu is off by K u mean|x| at most and x - mu by one rounding more; rstd by half the relative error of the variance, (2 K + 4) u, and two roundings."""
	x = x.double()
	dmu = (K + 2) * U * x.abs().mean(1, keepdim=True)
	xhat = (x - mu) * rstd
	drel = (K + 8) * U + dmu.square() * rstd.square()
	err = gamma.double().abs() * (dmu * rstd + xhat.abs() * drel) + 4 * U * (ref.abs() + (beta.double().abs() if beta is not None else 0))
	return err + half_step(ref.abs() + err, dtype)


PAIRS = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")]
WIDTHS = [1, 2, 7, 8, 9, 31, 64, 65, 128, 129, 255, 512, 513, 1000, 1024, 1025, 1280, 2048, 2049, 4096, 4097, 8192, 8193, 12289, 16383, 16384]


@pytest.mark.parametrize("xt,yt", PAIRS)
@pytest.mark.parametrize("E", WIDTHS)
def test_layernorm_forward(E, xt, yt):
	for rows, extra, shift, with_beta in ((1, 0, 0, True), (5, 3, 1, False), (67, 0, 0, True), (300, 8, 0, True)):
		g = gen(E * 7 + rows)
		x = Box(rows, E, TYPES[xt], extra, shift, normal(g, rows, E, scale=2.0, shift=0.5))
		y = Box(rows, E, TYPES[yt], extra, shift)
		gamma, beta = normal(g, E, shift=1.0), (normal(g, E) if with_beta else None)
		mean, rstd = torch.full((rows + 1,), 77.0, device=DEV), torch.full((rows + 1,), 77.0, device=DEV)
		ops.layernorm_stats_fwd(x.t, gamma, beta, y.t, mean[:rows], rstd[:rows], eps=1e-5)
		ref, mu, rs = ln_forward_ref(x.t, gamma, beta, 1e-5)
		near(y.t, ref, ln_forward_bound(x.t, gamma, beta, ref, mu, rs, TYPES[yt]), f"y {rows} x {E}")
		dmu = (K + 2) * U * x.t.double().abs().mean(1)
		near(mean[:rows], mu.squeeze(1), dmu, "mean")
		near(rstd[:rows], rs.squeeze(1), rs.squeeze(1) * ((K + 8) * U + dmu.square() * rs.squeeze(1).square()), "rstd")
		assert y.intact() and x.intact() and float(mean[rows]) == 77.0 and float(rstd[rows]) == 77.0
		y2 = Box(rows, E, TYPES[yt], extra, shift)
		ops.layernorm_stats_fwd(x.t, gamma, beta, y2.t)
		assert torch.equal(y2.buf, y.buf), "without statistics"


def ln_backward_ref(dy, x, gamma, mean, rstd, dx_in):
	dy, x, rstd = dy.double(), x.double(), rstd.double()[:, None]
	xhat = (x - mean.double()[:, None]) * rstd
	g = dy * gamma.double()
	dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
	dxhat = 2 * U * ((x.abs() + mean.double().abs()[:, None]) * rstd + xhat.abs())  # x - mean and its product with rstd
	err = rstd * (4 * U * g.abs() + (K + 4) * U * g.abs().mean(1, keepdim=True) + xhat.abs() * ((K + 6) * U * (g * xhat).abs().mean(1, keepdim=True) + (g.abs() * dxhat).mean(1, keepdim=True))
	              + dxhat * (g * xhat).mean(1, keepdim=True).abs())
	if dx_in is not None:
		dx = dx + dx_in.double()
	err = err + 4 * U * (dx.abs() + (dx_in.double().abs() if dx_in is not None else 0))
	return dx, err, (dy * xhat).sum(0), dy.sum(0), (dy.abs() * (xhat.abs() + dxhat)).sum(0), dy.abs().sum(0), (dy.abs() * dxhat).sum(0)


@pytest.mark.parametrize("xt,yt", PAIRS)
@pytest.mark.parametrize("E", WIDTHS)
def test_layernorm_backward(E, xt, yt):
	for rows, extra, shift, resid in ((1, 0, 0, True), (6, 3, 1, False), (131, 0, 0, True), (1500, 8, 0, False)):
		if rows * E > 6_000_000:
			rows = 6_000_000 // E
		g = gen(E * 5 + rows)
		x = Box(rows, E, TYPES[xt], extra, shift, normal(g, rows, E, scale=2.0, shift=0.5))
		dy = Box(rows, E, TYPES[yt], extra, shift, normal(g, rows, E))
		dx_in = Box(rows, E, TYPES[xt], extra, shift, normal(g, rows, E)) if resid else None
		dx = Box(rows, E, TYPES[xt], extra, shift)
		gamma = normal(g, E, shift=1.0)
		_, mu, rs = ln_forward_ref(x.t, gamma, None, 1e-5)
		mean, rstd = mu.squeeze(1).float(), rs.squeeze(1).float()
		dgamma, dbeta = torch.full((E,), 77.0, device=DEV), torch.full((E,), 77.0, device=DEV)
		ops.layernorm_stats_bwd(dy.t, x.t, gamma, mean, rstd, dx.t, dgamma, dbeta, dx_in=dx_in.t if resid else None)
		ref, err, rg, rb, ag, ab, xg = ln_backward_ref(dy.t, x.t, gamma, mean, rstd, dx_in.t if resid else None)
		near(dx.t, ref, err + half_step(ref.abs() + err, TYPES[xt]), f"dx {rows} x {E}")
		# a lane adds rows / (teams of the whole grid) <= 94 rows here (the fewest teams: 16 rows' worth for one block), then 16 teams, then 32 groups of at most 16 partial rows
		near(dgamma, rg, 160 * U * ag + xg, "dgamma")
		near(dbeta, rb, 160 * U * ab, "dbeta")
		assert dx.intact() and dy.intact() and x.intact()
		# the same bits again, alone and added to what is there
		again, more = torch.empty(E, device=DEV), dbeta.clone()
		dx2 = Box(rows, E, TYPES[xt], extra, shift)
		ops.layernorm_stats_bwd(dy.t, x.t, gamma, mean, rstd, dx2.t, again, None, dx_in=dx_in.t if resid else None)
		assert torch.equal(again, dgamma) and torch.equal(dx2.buf, dx.buf)
		ops.layernorm_stats_bwd(dy.t, x.t, gamma, mean, rstd, dx2.t, None, more, accumulate=True)
		assert torch.equal(more, dbeta + dbeta)


def test_layernorm_in_place():
	for E in (97, 509, 1280, 5001, 16384):
		for t in (F32, BF16):
			g = gen(E)
			x, dy, gamma, beta = normal(g, 40, E, dtype=t), normal(g, 40, E, dtype=t), normal(g, E), normal(g, E)
			y, dx = torch.empty_like(x), torch.empty_like(x)
			mean, rstd = torch.empty(40, device=DEV), torch.empty(40, device=DEV)
			ops.layernorm_stats_fwd(x, gamma, beta, y, mean, rstd)
			a = x.clone()
			ops.layernorm_stats_fwd(a, gamma, beta, a)
			assert torch.equal(a, y)
			ops.layernorm_stats_bwd(dy, x, gamma, mean, rstd, dx, dx_in=y)
			a = y.clone()
			ops.layernorm_stats_bwd(dy, x, gamma, mean, rstd, a, dx_in=a)
			assert torch.equal(a, dx)


def test_layernorm_no_rows_and_odd_values():
	gamma = torch.ones(33, device=DEV)
	none = torch.empty(0, 33, device=DEV)
	dgamma, dbeta, v = torch.full((33,), 5.0, device=DEV), torch.full((33,), 5.0, device=DEV), torch.empty(0, device=DEV)
	ops.layernorm_stats_fwd(none, gamma, None, none.clone(), v, v.clone())
	ops.layernorm_stats_bwd(none, none, gamma, v, v, none.clone(), dgamma, dbeta, accumulate=True)
	assert (dgamma == 5).all() and (dbeta == 5).all()
	ops.layernorm_stats_bwd(none, none, gamma, v, v, none.clone(), dgamma, dbeta)
	assert (dgamma == 0).all() and (dbeta == 0).all()
	# a row of equal values: variance 0; a NaN and an infinity stay in their own rows
	x = torch.ones(4, 33, device=DEV) * 3
	x[1, 32], x[2, 0] = float("nan"), float("inf")
	y = torch.empty_like(x)
	ops.layernorm_stats_fwd(x, gamma, None, y)
	assert (y[0] == 0).all() and (y[3] == 0).all() and y[1].isnan().all() and y[2].isnan().any()


def test_layernorm_beyond_32_bits():
	"""140 000 rows of 16 384: 2.3e9 elements."""
	rows, E = 140_000, 16384
	x = torch.empty(rows, E, dtype=BF16, device=DEV)
	last = normal(gen(3), 64, E, dtype=BF16)
	x.zero_()
	x[-64:] = last
	gamma, y = torch.ones(E, device=DEV), torch.empty_like(x)
	mean, rstd = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
	ops.layernorm_stats_fwd(x, gamma, None, y, mean, rstd)
	ref, mu, rs = ln_forward_ref(last, gamma, None, 1e-5)
	near(y[-64:], ref, ln_forward_bound(last, gamma, None, ref, mu, rs, BF16))
	dgamma = torch.empty(E, device=DEV)
	ops.layernorm_stats_bwd(x, x, gamma, mean, rstd, y, dgamma)
	dx, err, rg, _, ag, _, xg = ln_backward_ref(last, last, gamma, mean[-64:], rstd[-64:], None)
	near(y[-64:], dx, err + half_step(dx.abs() + err, BF16))
	near(dgamma, rg, 700 * U * ag + xg)  # 547 rows a block (zeros add exactly), 32 groups


# ---- dropout -------------------------------------------------------------------------------------------------------------------------------------------------------

def keep_ref(n, p, seed, site, step):
	"""The mask from the generator's definition, in numpy."""
	m, s = np.uint64(0xFFFFFFFF), np.uint64(32)
	b = np.arange((n + 7) // 8, dtype=np.uint64)
	c = [b & m, b >> s, np.full_like(b, site & 0xFFFFFFFF), np.full_like(b, step & 0xFFFFFFFF)]
	k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
	for _ in range(10):
		a, d = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
		c = [(d >> s) ^ c[1] ^ np.uint64(k0), d & m, (a >> s) ^ c[3] ^ np.uint64(k1), a & m]
		k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
	u = np.stack([h for w in c for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1).reshape(-1)[:n]
	return torch.from_numpy(u >= int(p * 65536 + 0.5)).to(DEV)


def test_philox_known_answers():
	"""The published test vectors of Philox4x32-10 (its authors' known-answer file: all zeros, all ones), through the mask's reference: the words' halves against thresholds."""
	def words(c, k):
		for _ in range(10):
			a, d = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
			c = [(d >> 32) ^ c[1] ^ k[0], d & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
			k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
		return c
	assert words([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
	assert words([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
	u = [h for w in words([0] * 4, [0] * 2) for h in (w & 0xFFFF, w >> 16)]
	for p in (0.2, 0.5, 0.77):
		x, y = torch.ones(1, 8, device=DEV), torch.empty(1, 8, device=DEV)
		ops.dropout_fwd(x, y, ops.Dropout(p, 0, 0))
		assert [v > 0 for v in y[0].tolist()] == [h >= int(p * 65536 + 0.5) for h in u]


@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("rows,cols,extra,shift", [(1, 1, 0, 0), (1, 7, 0, 1), (3, 8, 0, 0), (5, 13, 0, 1), (5, 13, 3, 1), (64, 512, 8, 0), (33, 509, 7, 0), (1, 100_001, 5, 0), (4099, 257, 0, 0), (5000, 3, 2, 0)])
def test_dropout(rows, cols, extra, shift, xt, yt):
	for p, seed, site, step in ((0.1, 0x1234567890ABCDEF, 3, None), (0.5, 5, 0xFFFFFFFF, 7), (0.0, 1, 1, 1), (1.0, 1, 1, 1), (0.999, 2 ** 64 - 1, 0, (1 << 32) + 9)):
		g = gen(rows + cols)
		x = Box(rows, cols, TYPES[xt], extra, shift, normal(g, rows, cols))
		r = Box(rows, cols, TYPES[yt], extra, shift, normal(g, rows, cols))
		y, z = Box(rows, cols, TYPES[yt], extra, shift), Box(rows, cols, TYPES[yt], extra, shift)
		drop, at = ops.Dropout(p, seed, site), None if step is None else torch.tensor(step, device=DEV)
		ops.dropout_fwd(x.t, y.t, drop, resid=r.t, step=at)
		ops.dropout_bwd(x.t, z.t, drop, step=at)
		keep = keep_ref(rows * cols, p, seed, site, step or 0).view(rows, cols)
		thr = int(p * 65536 + 0.5)
		ref = torch.where(keep, x.t.double() * (65536 / (65536 - thr) if thr < 65536 else 0.0), 0.0)
		assert torch.equal(z.t != 0, keep & (x.t != 0)) or yt == "f16"
		near(z.t, ref, 2 * U * ref.abs() + half_step(ref * (1 + 2 * U), TYPES[yt]), "dx")
		ref2 = ref + r.t.double()
		err = 3 * U * (ref.abs() + r.t.double().abs())
		near(y.t, ref2, err + half_step(ref2.abs() + err, TYPES[yt]), "y")
		assert y.intact() and z.intact()


def test_dropout_stops_what_it_drops_and_works_in_place():
	x = torch.full((64, 100), float("nan"), device=DEV)
	y = torch.empty_like(x)
	drop = ops.Dropout(0.3, 11, 4)
	ops.dropout_fwd(x, y, drop)
	keep = keep_ref(6400, 0.3, 11, 4, 0).view(64, 100)
	assert torch.equal(y.isnan(), keep) and (y[~keep] == 0).all()
	x = normal(gen(1), 64, 100)
	ops.dropout_fwd(x, y, drop, resid=x)
	a = x.clone()
	ops.dropout_fwd(a, a, drop, resid=a)
	assert torch.equal(a, y)
	for view in (x[:0], x[:, :0]):
		ops.dropout_fwd(view, view.clone(), drop)
	# the share of kept elements: 4 standard deviations of a binomial of 2^24 draws
	big = torch.ones(4096, 4096, device=DEV, dtype=BF16)
	out = torch.empty_like(big)
	ops.dropout_fwd(big, out, ops.Dropout(0.1, 99, 1))
	n, q = out.numel(), 1 - round(6553.6) / 65536
	assert abs(int((out != 0).sum()) - n * q) <= 4 * math.sqrt(n * q * (1 - q))


def test_dropout_beyond_32_bits():
	rows, cols = 140_000, 16384
	x = torch.ones(rows, cols, dtype=BF16, device=DEV)
	y = torch.empty_like(x)
	ops.dropout_fwd(x, y, ops.Dropout(0.5, 21, 2))
	n = rows * cols
	first = (n - 8 * 4096) // 8
	m, s = np.uint64(0xFFFFFFFF), np.uint64(32)
	b = np.arange(first, first + 4096, dtype=np.uint64)
	c, k0, k1 = [b & m, b >> s, np.full_like(b, 2), np.zeros_like(b)], 21, 0
	for _ in range(10):
		a, d = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
		c = [(d >> s) ^ c[1] ^ np.uint64(k0), d & m, (a >> s) ^ c[3] ^ np.uint64(k1), a & m]
		k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
	u = np.stack([h for w in c for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1).reshape(-1)
	assert torch.equal((y.view(-1)[-8 * 4096:] != 0).cpu(), torch.from_numpy(u >= 32768))


# ---- token rows ----------------------------------------------------------------------------------------------------------------------------------------------------

class Tokens:
	"""Logits in a wider buffer, targets, a padding mask with rows that leave a sequence empty, NaN logits where a position does not count."""

	def __init__(self, A, T, V, dtype, extra=0, shift=0, seed=0, tok=torch.int64, scale=3.0, empty=True, offsets=False):
		g = gen(seed + A * 31 + T * 7 + V)
		self.A, self.T, self.V, self.dtype, self.g = A, T, V, dtype, g
		self.box = Box(A * T, V, dtype, extra, shift, normal(g, A * T, V, scale=scale))
		self.logits = self.box.t
		if offsets:  # rows of negative numbers, rows of positive ones, rows of zeros of both signs, rows with most of the vocabulary masked out
			kind = torch.arange(A * T, device=DEV) % 5
			self.logits += torch.tensor([0.0, -60.0, 40.0, 0.0, 0.0], device=DEV)[kind].to(dtype)[:, None]
			self.logits[kind == 3] *= 0.0
			self.logits[3::5] = torch.where(torch.rand(self.logits[3::5].shape, generator=g, device=DEV) < 0.5, -0.0, 0.0).to(dtype)
			self.logits[4::5, 3:] = float("-inf")
		self.target = torch.randint(0, 3 if offsets else V, (A, T), generator=g, device=DEV).to(tok)
		length = torch.randint(1, T + 1, (A,), generator=g, device=DEV)
		if empty and A > 2:
			length[1] = 0
		self.pad = torch.arange(T, device=DEV)[None] >= length[:, None]
		self.valid = ~self.pad
		if T > 2 and A > 2:  # targets outside the vocabulary do not count either
			self.target[2, 0], self.target[2, 1] = -100 if tok == torch.int64 else -1, V
			self.valid = self.valid & (self.target >= 0) & (self.target < V)
		self.logits[~self.valid.view(-1)] = float("nan")
		x = torch.where(self.valid.view(-1, 1), self.logits.double(), torch.zeros((), device=DEV, dtype=torch.double))
		at = self.target.long().clamp(0, V - 1).view(-1, 1)
		self.lse = torch.logsumexp(x, 1)
		self.p = (x - self.lse[:, None]).exp()
		self.onehot = torch.zeros_like(x).scatter_(1, at, 1.0)
		self.d = (x - x.max(1, keepdim=True).values).abs().nan_to_num(posinf=0.0)  # (of a masked element: its exponential is a zero)
		# distance from the maximum: an exponential is off by that many u, relative
		self.lp = ((x.gather(1, at).squeeze(1) - self.lse).view(A, T) * self.valid).detach()
		# log s: K u for the sum, 4 u + the mean distance for the exponentials
		self.dlp = (U * (K + 4 + (self.p * self.d).sum(1).view(A, T)) + U * self.lp.abs()) * self.valid

	def dlogits(self, coef):
		c = (coef * self.valid).view(-1, 1)
		return c * (self.onehot - self.p)

	def dlogits_bound(self, coef, dcoef, ref, dtype):
		c, dc = (coef.abs() * self.valid).view(-1, 1), (dcoef * self.valid).view(-1, 1)
		err = dc * (self.onehot - self.p).abs() + c * U * (self.p * (K + 10 + self.d + (self.p * self.d).sum(1, keepdim=True)) + 2 * self.onehot)
		return err + half_step(ref.abs() + err, dtype)


def vocabularies(dtype):
	w = [1, 2, 5, 7, 8, 9, 64, 97, 255, 256, 257, 512, 513, 1024, 1025, 2048, 2056, 4097, 6911, 6912, 8192, 10007, 16384, 16391, 32768, 40001]
	return w + ([65544, 70001, 131072] if dtype != F32 else [32770, 65537])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_token_logprobs(dtype):
	for i, V in enumerate(vocabularies(dtype)):
		A, T, extra, shift, tok = ((5, 7, 0, 0, torch.int64), (3, 1, 3, 1, torch.int32), (4, 19, 8, 0, torch.int64))[i % 3]
		s = Tokens(A, T, V, dtype, extra, shift, tok=tok)
		out, lse = Box(A, T, F32, 2), torch.full((A * T + 1,), 77.0, device=DEV)
		ops.token_logprobs(s.logits, s.target, out.t, pad=s.pad, lse=lse[:A * T])
		near(out.t, s.lp, s.dlp, f"logp, V = {V}")
		near(lse[:A * T], s.lse * s.valid.view(-1), s.dlp.view(-1) + 2 * U * s.lse.abs(), f"lse, V = {V}")
		assert out.intact() and s.box.intact() and float(lse[-1]) == 77.0
		keep = torch.empty(A, T, device=DEV)
		ops.token_logprobs(s.logits, s.target, keep, pad=s.pad.to(torch.uint8))
		assert torch.equal(keep, out.t)
		# backward, a value for each token and one for each sequence, out of place and in place
		grad, dl = normal(s.g, A, T), Box(A * T, V, dtype, extra, shift)
		base = (s.lse.float() * s.valid.view(-1).float()).contiguous()
		for gr, full in ((grad, grad.double()), (grad[:, 0].contiguous(), grad[:, :1].double().expand(A, T))):
			ops.token_logprobs_bwd(s.logits, s.target, base, gr, dl.t, pad=s.pad)
			ref = s.dlogits(full)
			# lse as given is rounded: 1/2 step of itself, and x - lse rounds once more
			more = (full.abs() * s.valid).view(-1, 1) * s.p * U * (3 * s.lse.abs().view(-1, 1) + s.d)
			near(dl.t, ref, s.dlogits_bound(full, torch.zeros_like(full), ref, dtype) + more, f"dlogits, V = {V}")
			assert dl.intact()
		same = s.box.buf.clone()
		ops.token_logprobs_bwd(s.logits, s.target, base, gr, s.logits, pad=s.pad)
		assert torch.equal(s.logits, dl.t)
		s.box.buf.copy_(same)


def test_token_logprobs_odd_values():
	V = 300
	for dtype in (F32, BF16, F16):
		x = normal(gen(5), 6, V, dtype=dtype)
		low = torch.finfo(dtype).min
		x[0, 10:] = float("-inf")     # most of the vocabulary masked out
		x[1] = float("-inf")          # all of it
		x[2, 5] = float("inf")
		x[3, 7] = float("nan")
		x[4, 3:] = low                # masked with the type's lowest value
		t = torch.tensor([[0, 0, 0, 0, 1, 2]], device=DEV)
		out, lse = torch.empty(1, 6, device=DEV), torch.empty(6, device=DEV)
		ops.token_logprobs(x, t, out, lse=lse)
		ref = torch.log_softmax(x.double(), 1)
		want = ref[torch.arange(6, device=DEV), t[0]]
		assert out[0, 1:4].isnan().all() and torch.isfinite(out[0, [0, 4, 5]]).all()
		near(out[0, [0, 4, 5]], want[[0, 4, 5]], (K + 20) * U * (1 + want[[0, 4, 5]].abs()))
		x[5, 2] = float("-inf")       # the target itself is masked out
		ops.token_logprobs(x, t, out)
		assert float(out[0, 5]) == float("-inf")
		d = torch.empty_like(x)
		ops.token_logprobs_bwd(x, t, lse, torch.ones(1, 6, device=DEV), d)
		assert (d[0, 10:] == 0).all() and (d[4, 3:] == 0).all() and torch.isfinite(d[[0, 4, 5]]).all()
	# 70 001 columns: the form that reads a row twice sees the same values
	x = torch.full((3, 70001), float("-inf"), device=DEV)
	x[0, 60000], x[2, 69999], x[2, 3] = 2.0, 1.0, 1.0
	out = torch.empty(1, 3, device=DEV)
	ops.token_logprobs(x, torch.tensor([[60000, 5, 69999]], device=DEV), out)
	assert float(out[0, 0]) == 0.0 and math.isnan(float(out[0, 1])) and abs(float(out[0, 2]) + math.log(2)) < 1e-6


def test_token_logprobs_beyond_32_bits():
	"""17 000 rows of 131 072: 2.2e9 logits, of which a few rows at the end count."""
	A, T, V = 17_000, 1, 131072
	x = torch.empty(A, V, dtype=BF16, device=DEV)
	x[-5:] = normal(gen(9), 5, V, dtype=BF16)
	pad = torch.ones(A, 1, dtype=torch.bool, device=DEV)
	pad[-5:] = False
	t = torch.full((A, 1), V - 1, device=DEV)
	out, lse, d = torch.empty(A, 1, device=DEV), torch.empty(A, device=DEV), torch.full_like(x, 7)
	ops.token_logprobs(x, t, out, pad=pad, lse=lse)
	ops.token_logprobs_bwd(x, t, lse, torch.ones(A, device=DEV), d, pad=pad)
	ref = torch.log_softmax(x[-5:].double(), 1)
	near(out[-5:, 0], ref[:, -1], (K + 64) * U * (1 + ref[:, -1].abs()))
	assert (out[:-5] == 0).all() and not d[:-5].any()
	want = -ref.exp()
	want[:, -1] += 1
	near(d[-5:], want, half_step(want, BF16) + 256 * U * want.abs())


# ---- preference loss -----------------------------------------------------------------------------------------------------------------------------------------------

def pref_ref(z, beta, kind, e):
	if kind == "sigmoid":
		return -(1 - e) * torch.nn.functional.logsigmoid(z) - e * torch.nn.functional.logsigmoid(-z)
	return torch.relu(1 - z) if kind == "hinge" else ((z - 0.5) / beta) ** 2


PREF = [("sigmoid", 0.0, 0.1), ("sigmoid", 0.2, 0.5), ("hinge", 0.0, 0.3), ("square", 0.0, 0.2)]


@pytest.mark.parametrize("kind,e,beta", PREF)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,T,V,extra,shift", [(520, 7, 1000, 24, 0), (513, 3, 2500, 3, 1), (512, 12, 6912, 0, 0), (515, 2, 8191, 0, 0), (512, 32, 300, 0, 0), (512, 33, 300, 0, 0), (600, 2, 8200, 0, 0), (512, 5, 4097, 0, 0),
                                               (700, 40, 17, 0, 0), (1, 1, 5, 0, 0), (1, 1, 97, 3, 1), (3, 7, 257, 0, 0), (40, 7, 1000, 24, 0), (2, 130, 6912, 0, 0), (5, 12, 6911, 1, 0), (2, 4, 40001, 0, 0), (1, 3, 70001, 7, 0), (1500, 2, 33, 0, 0)])
def test_preference(n, T, V, extra, shift, dtype, kind, e, beta):
	s = Tokens(2 * n, T, V, dtype, extra, shift, tok=torch.int32 if n == 3 else torch.int64)
	ref = (s.lp + 0.7 * torch.randn(2 * n, T, generator=s.g, device=DEV, dtype=torch.double)).float()
	ref[~s.valid] = float("nan")  # not looked at
	weight = torch.rand(n, generator=s.g, device=DEV) + 0.5 if n % 2 else None
	if weight is not None and n > 2:
		weight[0] = 0.0
	scale = 3.0
	stats, margin, logp, dl = torch.empty(3, device=DEV), torch.empty(n, device=DEV), Box(2 * n, T, F32, 1), Box(2 * n * T, V, dtype, extra, shift)
	call = lambda **kw: ops.preference_loss(s.logits, s.target, ref, kw.pop("stats"), beta=beta, kind=kind, smoothing=e, pad=s.pad, weight=weight, grad_scale=scale, **kw)  # noqa: E731
	call(stats=stats, margin=margin, logp=logp.t, dlogits=dl.t)
	lp = s.lp.clone().requires_grad_()
	u = torch.where(s.valid, lp - torch.where(s.valid, ref.double(), 0.0), 0.0).sum(1)
	z = beta * (u[:n] - u[n:])
	w = torch.ones(n, device=DEV, dtype=torch.double) if weight is None else weight.double()
	each = pref_ref(z, beta, kind, e)
	loss = (w * each).sum() / w.sum()
	(coef,) = torch.autograd.grad(scale * loss, lp)
	dz = beta * (s.dlp.sum(1)[:n] + s.dlp.sum(1)[n:]) + U * z.detach().abs()
	curve = {"sigmoid": 0.25, "hinge": 0.0, "square": 2 / beta ** 2}[kind]  # the most that dl/dz changes with z
	if kind == "hinge" and bool(((z - 1).abs() <= dz).any()):
		pytest.skip("a margin within rounding of the hinge")
	dcoef = torch.cat([curve * dz * w, curve * dz * w])[:, None] / w.sum() * beta * scale + 6 * U * coef.abs()
	slope = torch.autograd.grad(pref_ref(zz := z.detach().requires_grad_(), beta, kind, e).sum(), zz)[0].abs()
	near(margin, z.detach(), dz, "margin")
	near(logp.t, s.lp, s.dlp, "logp")
	near(stats[0], loss.detach(), float((w * (slope * dz + curve * dz * dz)).sum() / w.sum() + 4 * U * loss.detach().abs()), "loss")
	near(stats[1], ((w * z).sum() / w.sum()).detach(), float((w * dz).sum() / w.sum() + 4 * U * z.detach().abs().max()), "mean margin")
	near(stats[2], w.sum(), float(2 * U * w.sum()), "weights")
	want = s.dlogits(coef)
	near(dl.t, want, s.dlogits_bound(coef, dcoef, want, dtype), "dlogits")
	assert dl.intact() and logp.intact() and s.box.intact()
	only = torch.empty(3, device=DEV)
	call(stats=only)
	assert torch.equal(only, stats)
	call(stats=only, dlogits=s.logits)  # in place
	assert torch.equal(s.logits, dl.t) and torch.equal(only, stats)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("op", ["logprob", "preference", "policy"])
@pytest.mark.parametrize("n,T,V", [(3000, 2, 17), (3000, 2, 100), (700, 5, 700), (520, 6, 1500), (600, 4, 3000), (520, 4, 6000), (30, 4, 6000), (20, 3, 9000), (4, 2, 70000)])
def test_rows_of_all_kinds(n, T, V, op, dtype):
	"""Rows whose numbers are all negative, all positive, zeros of both signs, or mostly masked out: gradients by every form of the kernels, at row counts that choose each."""
	A = 2 * n
	s = Tokens(A, T, V, dtype, offsets=True)
	old = torch.where(s.valid, s.lp - 0.1, 0.0).float()
	d = Box(A * T, V, dtype, 5, 1)
	adv = normal(s.g, A)
	if op == "logprob":
		lse, out = torch.empty(A * T, device=DEV), torch.empty(A, T, device=DEV)
		ops.token_logprobs(s.logits, s.target, out, pad=s.pad, lse=lse)
		near(out, s.lp, s.dlp, "logp")
		ops.token_logprobs_bwd(s.logits, s.target, lse, adv, d.t, pad=s.pad)
		coef = adv.double()[:, None].expand(A, T)
		dcoef = torch.zeros_like(coef)
		want = s.dlogits(coef)
		# lse rounds where it is kept, up to 70 here
		bound = s.dlogits_bound(coef, dcoef, want, dtype) + (coef.abs() * s.valid).reshape(-1, 1) * s.p * (U * (3 * s.lse.abs().view(-1, 1) + s.d) + s.dlp.view(-1, 1))
	elif op == "preference":
		stats = torch.empty(3, device=DEV)
		ops.preference_loss(s.logits, s.target, old, stats, beta=0.3, pad=s.pad, dlogits=d.t, grad_scale=float(n))
		u = torch.where(s.valid, s.lp - old.double(), 0.0).sum(1)
		z = 0.3 * (u[:n] - u[n:])
		c = -0.3 * torch.sigmoid(-z)
		coef = torch.cat([c, -c])[:, None].expand(A, T)
		dz = 0.3 * (s.dlp.sum(1)[:n] + s.dlp.sum(1)[n:])
		dcoef = torch.cat([dz, dz])[:, None].expand(A, T) * 0.3 * 0.25 + 8 * U * coef.abs()
		want = s.dlogits(coef)
		bound = s.dlogits_bound(coef, dcoef, want, dtype)
		near(stats[0], -torch.nn.functional.logsigmoid(z).mean(), float(dz.mean()) + 4 * U)
	else:
		stats = torch.empty(4, device=DEV)
		count = float(s.valid.sum())
		ops.policy_loss(s.logits, s.target, old, adv, stats, pad=s.pad, dlogits=d.t, grad_scale=count)
		q = torch.where(s.valid, (s.lp - old.double()).exp(), 0.0)  # 1.105: inside the clip range
		coef = -q * adv.double()[:, None]
		dcoef = coef.abs() * (s.dlp + 16 * U)
		want = s.dlogits(coef)
		bound = s.dlogits_bound(coef, dcoef, want, dtype)
	near(d.t, want, bound, f"dlogits of {op}")
	assert d.intact()


@pytest.mark.parametrize("dtype,n,T,V", [(F32, 512, 12, 6912), (BF16, 600, 3, 9000), (F16, 40, 20, 40000), (BF16, 600, 4, 3000), (F32, 600, 4, 200)])
def test_gradients_in_place_every_time(dtype, n, T, V):
	"""The gradient written over its logits has the bits of the one written beside them, twenty times over: the target's logit is read before anything may be stored there."""
	s = Tokens(2 * n, T, V, dtype)
	old, adv = s.lp.float(), normal(s.g, 2 * n)
	keep, d = s.logits.clone(), torch.empty(2 * n * T, V, device=DEV, dtype=dtype)
	st, st4, lse = torch.empty(3, device=DEV), torch.empty(4, device=DEV), (s.lse * s.valid.view(-1)).float()
	for call in (lambda o: ops.preference_loss(s.logits, s.target, old, st, beta=0.2, pad=s.pad, dlogits=o), lambda o: ops.policy_loss(s.logits, s.target, old, adv, st4, pad=s.pad, dlogits=o),
	             lambda o: ops.token_logprobs_bwd(s.logits, s.target, lse, adv, o, pad=s.pad)):
		call(d)
		for _ in range(20):
			s.logits.copy_(keep)
			call(s.logits)
			assert torch.equal(s.logits, d)
		s.logits.copy_(keep)


def test_preference_without_weight_or_tokens():
	s = Tokens(6, 4, 50, BF16)
	ref, stats, d = torch.zeros(6, 4, device=DEV), torch.full((3,), 7.0, device=DEV), torch.full((24, 50), 7.0, device=DEV, dtype=BF16)
	ops.preference_loss(s.logits, s.target, ref, stats, beta=0.1, pad=s.pad, weight=torch.zeros(3, device=DEV), dlogits=d)
	assert stats.tolist() == [0.0, 0.0, 0.0] and not d.any()
	d.fill_(7)
	ops.preference_loss(s.logits, s.target, ref, stats, beta=0.1, pad=torch.ones_like(s.pad), dlogits=d)
	assert abs(float(stats[0]) - math.log(2)) < 2 * U and float(stats[1]) == 0 and float(stats[2]) == 3 and not d.any()


# ---- policy loss ---------------------------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("per_seq", [False, True])
@pytest.mark.parametrize("kl,adv_dim", [(0.0, 1), (0.1, 2)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("A,T,V,extra,shift", [(1, 1, 5, 0, 0), (1, 1, 97, 3, 1), (7, 7, 257, 0, 0), (80, 7, 1000, 24, 0), (5, 130, 6912, 0, 0), (9, 12, 6911, 1, 0), (4, 4, 40001, 0, 0), (3, 3, 70001, 7, 0), (3000, 2, 33, 0, 0)])
def test_policy(A, T, V, extra, shift, dtype, kl, adv_dim, per_seq):
	lo, hi, scale = 0.2, 0.3, 5.0
	s = Tokens(A, T, V, dtype, extra, shift)
	noise = lambda sd: sd * torch.randn(A, T, generator=s.g, device=DEV, dtype=torch.double)  # noqa: E731
	d = noise(0.3)
	for end in (math.log(1 - lo), math.log(1 + hi)):  # (a ratio within rounding of a border may fall on either side of it)
		d = torch.where((d - end).abs() < 1e-3, d + 5e-3, d)
	nan = torch.full((), float("nan"), device=DEV, dtype=torch.double)
	old = torch.where(s.valid, s.lp - d, nan).float()
	ref = torch.where(s.valid, s.lp + noise(0.4), nan).float() if kl else None
	adv = normal(s.g, A) if adv_dim == 1 else torch.where(s.valid, noise(1.0), nan).float()
	stats, logp, dl = torch.empty(4, device=DEV), Box(A, T, F32, 1), Box(A * T, V, dtype, extra, shift)
	call = lambda **kw: ops.policy_loss(s.logits, s.target, old, adv, kw.pop("stats"), clip=(lo, hi), ref=ref, kl_coef=kl, per_sequence=per_seq, pad=s.pad, grad_scale=scale, **kw)  # noqa: E731
	call(stats=stats, logp=logp.t, dlogits=dl.t)
	zero = torch.zeros((), device=DEV, dtype=torch.double)
	clean = lambda t: torch.where(s.valid, t.double(), zero)  # noqa: E731
	lp = s.lp.clone().requires_grad_()
	q, a = (lp - clean(old)).exp(), clean(adv if adv_dim == 2 else adv[:, None].expand(A, T))
	held = q.clamp(1 - lo, 1 + hi)
	each = -torch.minimum(q * a, held * a)
	term = torch.zeros_like(q)
	if kl:
		dd = clean(ref) - lp
		term = torch.expm1(dd) - dd
		each = each + kl * term
	n = s.valid.sum()
	share = s.valid.double() / n.clamp(min=1)
	if per_seq:
		share = s.valid.double() / s.valid.sum(1, keepdim=True).clamp(min=1) / s.valid.any(1).sum().clamp(min=1)
	loss = (each * share).sum()
	(coef,) = torch.autograd.grad(scale * loss, lp)
	cut = ((q * a > held * a) & s.valid).double().detach()
	# q and exp(d): off by the error of lp and four roundings; each enters the gradient with a factor |a| or kl
	dq = s.dlp + 8 * U
	dcoef = share * scale * (a.abs() * q.detach() * dq + kl * (term.detach() + (dd.detach().exp() if kl else 0)) * dq) + 8 * U * coef.abs() + share * scale * 8 * U * (a.abs() * q.detach() + kl)
	dloss = float((share * ((a.abs() * q.detach()) * dq + kl * (dd.detach().exp() if kl else 0) * dq + 8 * U * each.detach().abs())).sum())
	near(logp.t, s.lp, s.dlp, "logp")
	near(stats[0], loss.detach(), dloss + 2 * U * float(loss.detach().abs()), "loss")
	near(stats[1], (term * share).sum().detach(), float((share * (torch.expm1(dd.detach()).abs() * dq if kl else 0 * share) + 4 * U * share * term.detach()).sum()), "kl")
	near(stats[2], (cut * share).sum(), 4 * U, "clipped")
	assert float(stats[3]) == float(n)
	want = s.dlogits(coef)
	near(dl.t, want, s.dlogits_bound(coef, dcoef, want, dtype), "dlogits")
	assert dl.intact() and logp.intact() and s.box.intact()
	only = torch.empty(4, device=DEV)
	call(stats=only)
	assert torch.equal(only, stats)
	call(stats=only, dlogits=s.logits)
	assert torch.equal(s.logits, dl.t) and torch.equal(only, stats)


def test_policy_no_counted_row():
	s = Tokens(6, 4, 50, BF16)
	f, stats, d = torch.full((6, 4), float("nan"), device=DEV), torch.full((4,), 7.0, device=DEV), torch.full((24, 50), 7.0, device=DEV, dtype=BF16)
	for per_seq in (False, True):
		ops.policy_loss(s.logits, s.target, f, f, stats.fill_(7), ref=f, kl_coef=0.1, per_sequence=per_seq, pad=torch.ones_like(s.pad), dlogits=d.fill_(7), logp=(lp := torch.full((6, 4), 7.0, device=DEV)))
		assert not stats.any() and not d.any() and not lp.any()


@pytest.mark.parametrize("which", ["preference", "policy"])
def test_gradient_against_differences(which):
	"""Central differences of the kernels' own loss along a direction v: the truncation is h^2 / 6 of a third derivative of at most ~10 |grad| per unit of v, each loss is off by
	2 u of itself and what its log-probabilities are off by (less than 100 u a token, a share of 1 / tokens each, times at most 2)."""
	A, T, V, h = 8, 5, 300, 1e-2
	s = Tokens(A, T, V, F32, scale=1.5)
	old = torch.where(s.valid, s.lp + 0.05 * torch.randn(A, T, generator=s.g, device=DEV), 0.0).float()
	adv = normal(s.g, A)

	def loss(x, d=None):
		st = torch.empty(3 if which == "preference" else 4, device=DEV)
		if which == "preference":
			ops.preference_loss(x, s.target, old, st, beta=0.5, smoothing=0.1, pad=s.pad, dlogits=d)
		else:
			ops.policy_loss(x, s.target, old, adv, st, clip=(0.5, 0.9), ref=old, kl_coef=0.2, pad=s.pad, dlogits=d)
		return float(st[0])
	d = torch.empty(A * T, V, device=DEV)
	base = loss(s.logits, d)
	for k in range(4):
		v = torch.randn(A * T, V, generator=s.g, device=DEV)
		v[~s.valid.view(-1)] = 0
		want = float((d.double() * v.double()).sum())
		got = (loss(s.logits + h * v) - loss(s.logits - h * v)) / (2 * h)
		size = float((d.abs() * v.abs()).sum())
		assert abs(got - want) <= 10 * h * h / 6 * size * 10 + (2 * abs(base) + 400) * U / h, (got, want)


# ---- refusals that need device tensors, streams, graphs, together ---------------------------------------------------------------------------------------------------

def test_refusals():
	f, h = torch.zeros(6, 8, device=DEV), torch.zeros(6, 8, device=DEV, dtype=BF16)
	e, v6, i = torch.zeros(8, device=DEV), torch.zeros(6, device=DEV), torch.zeros(2, 3, device=DEV, dtype=torch.int64)
	r, st = torch.zeros(2, 3, device=DEV), torch.zeros(4, device=DEV)
	o = torch.zeros(6, 8, device=DEV)
	value = [lambda: ops.layernorm_stats_fwd(f.t(), v6, None, o.t()), lambda: ops.layernorm_stats_fwd(f, e, None, o[:5]), lambda: ops.layernorm_stats_fwd(f, e[:7], None, o),
	         lambda: ops.layernorm_stats_fwd(f, e, None, o, v6[:5]), lambda: ops.layernorm_stats_fwd(f[0], e, None, o), lambda: ops.layernorm_stats_fwd(f, e, None, o.view(-1)[1:41].view(5, 8)),
	         lambda: ops.layernorm_stats_fwd(f[:1].expand(6, 8), e, None, o), 
	         lambda: ops.layernorm_stats_fwd(torch.zeros(1, 16385, device=DEV), torch.zeros(16385, device=DEV), None, torch.zeros(1, 16385, device=DEV)),
	         lambda: ops.layernorm_stats_bwd(f, f, e, v6, v6, o, e.clone(), dx_in=f[:5]),
	         	         lambda: ops.dropout_fwd(f, o, ops.Dropout(1.5)), lambda: ops.dropout_fwd(f, o, ops.Dropout(float("nan"))), lambda: ops.dropout_fwd(f, o, ops.Dropout(0.1), resid=o[:5]),
	         lambda: ops.dropout_fwd(f, o, ops.Dropout(0.1), step=torch.zeros(2, dtype=torch.int64, device=DEV)), 
	         lambda: ops.token_logprobs(f[:5], i, r), lambda: ops.token_logprobs(f, i, r[:, :2]), lambda: ops.token_logprobs(f, i, r, pad=torch.zeros(3, 2, device=DEV, dtype=torch.bool)),
	         lambda: ops.token_logprobs(f[:, :0], i, r), lambda: ops.token_logprobs_bwd(f, i, v6, v6[:3], o),
	         lambda: ops.preference_loss(f[:3], i[:1], r[:1], st[:3], beta=0.1), lambda: ops.preference_loss(f, i, r, st, beta=0.1), lambda: ops.preference_loss(f, i, r, st[:3], beta=0.0),
	         lambda: ops.preference_loss(f, i, r, st[:3], beta=0.1, kind="other"), lambda: ops.preference_loss(f, i, r, st[:3], beta=0.1, kind="hinge", smoothing=0.1),
	         lambda: ops.preference_loss(f, i, r, st[:3], beta=0.1, weight=v6[:2]), lambda: ops.preference_loss(f[:0], i[:0], r[:0], st[:3], beta=0.1),
	         lambda: ops.policy_loss(f, i, r, v6[:2], st, clip=(1.5, 0.2)), lambda: ops.policy_loss(f, i, r, v6[:2], st, kl_coef=-1.0), lambda: ops.policy_loss(f, i, r, v6[:3], st),
	         lambda: ops.policy_loss(f[:0], i[:0], r[:0], v6[:0], st)]
	for k, call in enumerate(value):
		with pytest.raises(ValueError):
			call()
			print("accepted:", k)
	kind = [lambda: ops.layernorm_stats_fwd(h, e, None, o), lambda: ops.layernorm_stats_fwd(h, e, None, h.to(F16)), lambda: ops.layernorm_stats_fwd(f, e.to(BF16), None, o),
	        lambda: ops.layernorm_stats_fwd(f.double(), e, None, o), lambda: ops.layernorm_stats_bwd(f, f, e, v6, v6, h), lambda: ops.layernorm_stats_bwd(f, h, e, v6, v6, h.clone()),
	        lambda: ops.dropout_fwd(h, h.to(F16), ops.Dropout(0.1)), lambda: ops.dropout_fwd(f, o, ops.Dropout(0.1), resid=h),
	        lambda: ops.dropout_fwd(f, o, ops.Dropout(0.1), step=torch.zeros(1, dtype=torch.int32, device=DEV)), lambda: ops.token_logprobs(f, i.float(), r), lambda: ops.token_logprobs(f, i, r.double()),
	        lambda: ops.token_logprobs_bwd(f, i, v6, v6[:2].double(), o), lambda: ops.token_logprobs_bwd(f, i, v6, v6[:2].contiguous(), h), lambda: ops.policy_loss(f, i, r, None, st)]
	for k, call in enumerate(kind):
		with pytest.raises(TypeError):
			call()
			print("accepted:", k)
	overlap = [lambda: ops.layernorm_stats_fwd(f[:3], e, None, f[1:4]), lambda: ops.layernorm_stats_fwd(f, e, None, f.view(BF16)[:, :8]),
	           lambda: ops.layernorm_stats_bwd(f, f, e, v6, v6, o, (same := e.clone()), same), lambda: ops.layernorm_stats_bwd(f, f, e, v6, v6.clone(), o, e),
	           lambda: ops.dropout_fwd(f[:3], f[2:5], ops.Dropout(0.1)), lambda: ops.token_logprobs(f, i, f.view(-1)[:6].view(2, 3)), lambda: ops.layernorm_stats_fwd(f, e.cpu(), None, o),
	           lambda: ops.policy_loss(f, i, r, v6[:2], st, logp=r), lambda: ops.preference_loss(f, i, r, st[:3], beta=0.1, margin=st[2:3])]
	for k, call in enumerate(overlap):
		with pytest.raises(_lib.NovicHipError):
			call()
			print("accepted:", k)


class Step:
	"""A fine-tuning step of one block and the output layer: h -> dropout + residual -> LayerNorm -> logits -> loss -> back to h, the weights and the norm's affine parameters."""

	def __init__(self, which, seed, n=24, T=7, E=512, V=1000):
		g = gen(seed)
		self.which, self.n, self.T, self.E, self.V = which, n, T, E, V
		A, M, Vs = 2 * n, 2 * n * T, (V + 63) // 64 * 64
		self.s = Tokens(A, T, V, BF16, seed=seed)
		self.h, self.resid = normal(g, M, E, dtype=BF16), normal(g, M, E)
		self.gamma, self.beta = normal(g, E, scale=0.1, shift=1.0), normal(g, E, scale=0.1)
		self.w = torch.zeros(Vs, E, device=DEV, dtype=BF16)
		self.w[:V] = normal(g, V, E, scale=0.06)
		self.wt = self.w.t().contiguous()
		self.old = torch.where(self.s.valid, -7.0 + 0.3 * torch.randn(A, T, generator=g, device=DEV), 0.0)
		self.adv = normal(g, A)
		self.step = torch.zeros((), dtype=torch.int64, device=DEV)
		z = lambda *shape, dtype=F32: torch.zeros(*shape, device=DEV, dtype=dtype)  # noqa: E731
		self.x, self.y, self.mean, self.rstd = z(M, E), z(M, E, dtype=BF16), z(M), z(M)
		self.logits, self.dlogits, self.dy = z(M, Vs, dtype=BF16), z(M, Vs, dtype=BF16), z(M, E, dtype=BF16)
		self.dw, self.dx, self.dh, self.dgamma, self.dbeta = z(Vs, E), z(M, E), z(M, E, dtype=BF16), z(E), z(E)
		self.stats, self.drop = z(3 if which == "preference" else 4), ops.Dropout(0.1, 77, 5)

	def run(self):
		s, M, Vs = self.s, self.x.shape[0], self.w.shape[0]
		ops.dropout_fwd(self.h, self.x, self.drop, resid=self.resid, step=self.step)
		ops.layernorm_stats_fwd(self.x, self.gamma, self.beta, self.y, self.mean, self.rstd)
		ops.gemm(self.y, self.w, M, Vs, self.E, out=self.logits)
		if self.which == "preference":
			ops.preference_loss(self.logits[:, :self.V], s.target, self.old, self.stats, beta=0.1, pad=s.pad, dlogits=self.dlogits[:, :self.V])
		else:
			ops.policy_loss(self.logits[:, :self.V], s.target, self.old, self.adv, self.stats, ref=self.old, kl_coef=0.1, pad=s.pad, dlogits=self.dlogits[:, :self.V])
		ops.gemm(self.dlogits, self.wt, M, self.E, Vs, out=self.dy)
		self.dw.zero_()
		ops.gemm(self.dlogits, self.y, Vs, self.E, M, a_kstrided=True, b_kstrided=True, kind=ops.EPI_ATOMIC_F32, out=self.dw, ldc=self.E)
		ops.layernorm_stats_bwd(self.dy, self.x, self.gamma, self.mean, self.rstd, self.dx, self.dgamma, self.dbeta)
		ops.dropout_bwd(self.dx, self.dh, self.drop, step=self.step)
		self.step += 1
		return [t.clone() for t in (self.stats, self.dh, self.dx, self.dw, self.dgamma, self.dbeta)]

	def reference(self, step):
		"""The same in 64 bits, by autograd over the definitions (on the host: the wide products need no device)."""
		c = lambda t: t.detach().cpu().double()  # noqa: E731
		s, n, T, V = self.s, self.n, self.T, self.V
		h, resid, gamma, beta, w = (c(t).requires_grad_() for t in (self.h, self.resid, self.gamma, self.beta, self.w[:V]))
		keep = keep_ref(h.numel(), 0.1, 77, 5, step).view_as(self.h).cpu()
		x = resid + torch.where(keep, h * (65536 / (65536 - 6554)), 0.0)
		mu = x.mean(1, keepdim=True)
		y = (x - mu) * ((x - mu).square().mean(1, keepdim=True) + 1e-5).rsqrt() * gamma + beta
		valid = s.valid.cpu()
		lp = torch.log_softmax(y @ w.t(), 1).gather(1, s.target.cpu().clamp(0, V - 1).view(-1, 1)).view(2 * n, T)
		old = c(self.old)
		if self.which == "preference":
			u = torch.where(valid, lp - old, 0.0).sum(1)
			z = 0.1 * (u[:n] - u[n:])
			loss = -torch.nn.functional.logsigmoid(z).mean()
		else:
			q, a = (lp - old).exp(), c(self.adv)[:, None]
			each = -torch.minimum(q * a, q.clamp(0.8, 1.2) * a) + 0.1 * (torch.expm1(old - lp) - (old - lp))
			loss = torch.where(valid, each, 0.0).sum() / valid.sum()
		return loss.detach(), torch.autograd.grad(loss, (h, resid, w, gamma, beta))


@pytest.mark.parametrize("which", ["preference", "policy"])
def test_together(which):
	"""Against 64 bits.  Between the operators stand five roundings to bf16 (the normalised rows, the logits, dlogits, dy, dh: 2^-9 each on average, 2^-8 at most) and the products'
	own; a logit of size 4 is off by 2^-7 at most, which its probability is then off by, relative: 2-norms within 5 * 2^-8 + 2^-7 < 0.03.  A policy ratio within 2^-6 of a border
	of the clip range may fall on the other side of it: such rows are kept out of the comparison by their own gradients' 2-norm (see the choice of `old`: sd 0.3 around -7 puts
	ratios everywhere), so the policy form is compared with ratios as the kernel's own log-probabilities give them."""
	st = Step(which, 3)
	if which == "policy":  # ratios well inside or outside the clip range, by the decoder's own log-probabilities
		st.run()
		lp = torch.empty(2 * st.n, st.T, device=DEV)
		ops.token_logprobs(st.logits[:, :st.V], st.s.target, lp, pad=st.s.pad)
		st.step.zero_()
		g = gen(8)
		d = torch.where(torch.rand(lp.shape, generator=g, device=DEV) < 0.3, 0.4, 0.08) * torch.where(torch.rand(lp.shape, generator=g, device=DEV) < 0.5, -1.0, 1.0)
		st.old = (lp - d).masked_fill(~st.s.valid, 0.0)
	got = st.run()
	loss, grads = st.reference(0)
	assert abs(float(got[0][0]) - float(loss)) <= 0.03 * max(1.0, abs(float(loss)))
	for name, a, b in zip(("dh", "dx", "dw", "dgamma", "dbeta"), (got[1], got[2], got[3][:st.V], got[4], got[5]), grads):
		rel = float((a.cpu().double() - b).norm() / b.norm())
		assert rel <= 0.03, f"{name}: {rel}"
	assert not got[3][st.V:].any()  # the padded columns of the logits' gradient stayed zeros


def test_captured_and_replayed():
	"""Two steps captured in graphs of their own, replayed in turn and at the same time on two streams, with eager work between: each replay equals the eager pass of its step
	counter.  (The weight gradient's atomics are compared to 2^-10 of its largest value.)"""
	eager = {w: [r.run() for _ in range(4)] for w, r in ((w, Step(w, 3)) for w in ("preference", "policy"))}

	def same(a, b):
		for k, (x, y) in enumerate(zip(a, b)):
			if k == 3:
				assert float((x - y).abs().max()) <= float(y.abs().max()) * 2 ** -10
			else:
				assert torch.equal(x, y), k
	graphs = {}
	for w in ("preference", "policy"):
		st = Step(w, 3)
		st.run()
		st.step.zero_()
		torch.cuda.synchronize()
		graph = torch.cuda.CUDAGraph()
		with ops.graph_capture(graph, ops.capture_stream(DEV)):
			out = st.run()
		graphs[w] = (st, graph, out)
	lanes = ops.lane_streams(DEV, 2)
	for k in range(4):
		junk = Step("policy", 11, n=5)
		for (w, (st, graph, out)), lane in zip(graphs.items(), lanes):
			lane.wait_stream(torch.cuda.current_stream())
			with torch.cuda.stream(lane):
				graph.replay()
		junk.run()  # eager work beside the replays
		torch.cuda.synchronize()
		for w, (st, graph, out) in graphs.items():
			same(out, eager[w][k])
	ops.retire_graphs([g for _, g, _ in graphs.values()])


def test_two_streams_at_once():
	"""The same calls on two streams, with inputs of their own: each call's workspace is its own."""
	eager = [Step("preference", k, n=40).run() for k in (1, 2)]
	steps = [Step("preference", k, n=40) for k in (1, 2)]
	torch.cuda.synchronize()
	got = [None, None]
	for _ in range(5):
		for k, lane in enumerate(ops.lane_streams(DEV, 2)):
			with torch.cuda.stream(lane):
				steps[k].step.zero_()
				got[k] = steps[k].run()
	torch.cuda.synchronize()
	for a, b in zip(got, eager):
		for k, (x, y) in enumerate(zip(a, b)):
			assert torch.equal(x, y) if k != 3 else float((x - y).abs().max()) <= float(y.abs().max()) * 2 ** -10


# ---- logits so large that their product with log2 e rounds by whole exponents, or is no number: rows that a mask of -1e10, -1e30 or the type's lowest value leaves empty ------------

def far_rows(n, V, dtype):
	"""n rows of V logits and a target for each, near a level c: all c; all c but the target, which is c / 2; c with two at c / 2, one of them the target; c with ordinary logits in front."""
	top = torch.finfo(dtype).max
	levels = [c for c in (-top, -1e30, -1e10, -1.5e9, -1.3e9, -1e9, -3e4, 3e4, 1e9, 1.3e9, 1.5e9, 1e10, 1e30, top) if abs(c) <= top]
	r = torch.arange(n, device=DEV)
	c = torch.tensor(levels, dtype=torch.double, device=DEV)[r % len(levels)].to(dtype)
	kind = r // len(levels) % 4
	target = (r * 7919 + 3) % V
	x = c[:, None].repeat(1, V)
	half = (c.double() / 2).to(dtype)
	neg = c < 0
	for k in (1, 2):
		pick = (kind == k) & neg  # (with c > 0 the rest would be larger by more than fp32 holds)
		x[pick, target[pick]] = half[pick]
		if k == 2:
			x[pick, (target[pick] + 1) % V] = half[pick]
	few = min(3, V)
	pick = (kind == 3) & neg
	x[pick, :few] = normal(gen(V), n, few, dtype=dtype)[pick]
	target[pick] = target[pick] % few
	ref = torch.log_softmax(x.double(), 1)
	lp = ref.gather(1, target[:, None]).squeeze(1)
	# The sum is seen from M = fl(m log2 e), up to 2^-24 |M| from the maximum (|M| <= 2.1e9, beyond which m itself is the point): that far is every exponent, its rounding and that of
	# log2 e are u relative each
	m = x.double().abs().amax(1).clamp(max=2.1e9)
	return x, target, ref.exp(), lp, U * (K + 8 + lp.abs() + 4 * 2.0 ** -24 * 1.45 * m)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [5, 130, 500, 900, 1500, 5000, 10007, 20001, 70001])
def test_far_logits(V, dtype):
	A, T = 8, 14
	x, target, p, lp, bound = far_rows(A * T, V, dtype)
	target = target.view(A, T)
	out, lse = torch.empty(A, T, device=DEV), torch.empty(A * T, device=DEV)
	ops.token_logprobs(x, target, out, lse=lse)
	near(out, lp.view(A, T), bound.view(A, T), f"logp, V = {V}")
	want = torch.logsumexp(x.double(), 1)
	near(lse, want.float().double(), bound + 2 * U * want.abs(), "lse")
	onehot = torch.zeros_like(p).scatter_(1, target.view(-1, 1), 1.0)
	stats, d = torch.empty(4, device=DEV), torch.empty_like(x)
	ops.policy_loss(x, target, out, torch.full((A,), -float(A * T), device=DEV), stats, dlogits=d)  # ratio 1: the gradient of the sum of the log-probabilities, negated
	ref = onehot - p
	near(d, ref, bound[:, None] * (p + onehot) * 3 + half_step(ref, dtype), f"policy gradient, V = {V}")
	assert abs(float(stats[0]) - A * T) <= 1e-4 * A * T
	stats, d, n = torch.empty(3, device=DEV), torch.empty_like(x), A // 2
	margin = torch.empty(n, device=DEV)
	ops.preference_loss(x, target, out, stats, beta=2.0 * n, kind="square", margin=margin, dlogits=d)  # margin 0: slope -1 / beta^2, n of them, times beta
	ref = torch.cat([-(onehot - p)[:n * T], (onehot - p)[n * T:]]) / (2.0 * n * n)
	near(d, ref, bound[:, None] * (p + onehot) / (2.0 * n * n) * 4 + float(margin.abs().max()) * (p + onehot) / n + half_step(ref, dtype), f"preference gradient, V = {V}")
	assert abs(float(stats[1])) <= 2 * n * 2 * T * U * float(lp.abs().max()) + 1e-30


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [600, 4000])
def test_far_logits_pair_by_pair(V, dtype):
	n, T = 560, 3
	x, target, p, lp, bound = far_rows(2 * n * T, V, dtype)
	target = target.view(2 * n, T)
	ref, out, stats, margin, d = lp.float().view(2 * n, T), torch.empty(2 * n, T, device=DEV), torch.empty(3, device=DEV), torch.empty(n, device=DEV), torch.empty_like(x)
	ops.preference_loss(x, target, ref, stats, beta=1.0, kind="hinge", logp=out, margin=margin, dlogits=d)
	near(out, lp.view(2 * n, T), bound.view(2 * n, T))
	onehot = torch.zeros_like(p).scatter_(1, target.view(-1, 1), 1.0)
	near(margin, torch.zeros(n, device=DEV, dtype=torch.double), (2 * bound + U * lp.abs()).view(2, n, T).sum((0, 2)))
	want = torch.cat([-(onehot - p)[:n * T], (onehot - p)[n * T:]]) / n  # every margin is below 1
	near(d, want, bound[:, None] * (p + onehot) / n * 4 + half_step(want, dtype), "gradient")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,T,V", [(513, 9, 5000), (512, 20, 3000), (515, 32, 4001), (512, 8, 4096), (512, 9, 8192)])
def test_preference_many_long_rows(n, T, V, dtype):
	"""Pairs of more long rows than their workgroup has waves."""
	test_preference(n, T, V, 3, 1, dtype, "sigmoid", 0.1, 0.3)


def test_counts_beyond_their_types_are_refused():
	"""Row and column counts that a C int does not hold are refused, not cut to their low 32 bits."""
	x = torch.empty((1 << 32) + 5, 1, dtype=BF16, device=DEV)
	one = torch.ones(1, device=DEV)
	with pytest.raises(ValueError):
		ops.layernorm_stats_fwd(x, one, None, x)
	with pytest.raises(ValueError):
		ops.layernorm_stats_bwd(x, x, one, torch.empty(5, device=DEV), torch.empty(5, device=DEV), x)
	row, t = x.view(1, -1), torch.zeros(1, 1, dtype=torch.int64, device=DEV)
	with pytest.raises(ValueError):
		ops.token_logprobs(row, t, torch.empty(1, 1, device=DEV))
	with pytest.raises(ValueError):
		ops.preference_loss(torch.zeros(2, 4, device=DEV), t.repeat(2, 1), torch.zeros(2, 1, device=DEV), torch.empty(3, device=DEV), beta=float("inf"))
