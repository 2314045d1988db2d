"""The operators of decoder fine-tuning, case by case: LayerNorm with kept statistics, counter-based dropout, token log-probabilities, the preference loss and the
clipped policy loss.  Each in its plain form (elementary torch operations) and, where `own` is true, as a program calls it through novic_amd.ops."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def listed():
	return [
		# LayerNorm of the decoder's training step: 8192 labels x 7 positions, the fp32 residual stream to the bf16 operand of a matrix product
		{"name": "norm_fwd_step", "op": "norm", "dir": "fwd", "rows": 57344, "cols": 512, "x": "f32", "y": "bf16", "beta": False, "resid": False},
		# an image tower's block in fine-tuning (256 images x 257 tokens, width 1280): both affine gradients and the residual branch's gradient added
		{"name": "norm_bwd_tower", "op": "norm", "dir": "bwd", "rows": 65792, "cols": 1280, "x": "bf16", "y": "bf16", "beta": True, "resid": True},
		# an odd width in half precision: no row starts on a vector boundary
		{"name": "norm_bwd_odd", "op": "norm", "dir": "bwd", "rows": 1021, "cols": 509, "x": "f16", "y": "f16", "beta": True, "resid": False},
		# a micro-batch of 16 labels in a smoke run: launch latency
		{"name": "norm_bwd_small", "op": "norm", "dir": "bwd", "rows": 16, "cols": 512, "x": "f32", "y": "bf16", "beta": False, "resid": True},
		# the exit of a sublayer in the training step: bf16 branch, dropped out and added to the fp32 residual stream
		{"name": "dropout_fwd_step", "op": "dropout", "dir": "fwd", "rows": 57344, "cols": 512, "x": "bf16", "y": "f32", "resid": True, "p": 0.1},
		# its backward pass on a small odd matrix in single precision
		{"name": "dropout_bwd_odd", "op": "dropout", "dir": "bwd", "rows": 257, "cols": 1153, "x": "f32", "y": "f32", "resid": False, "p": 0.25},
		# candidate labels of one small batch scored under a frozen decoder
		{"name": "logprob_fwd_small", "op": "logprob", "dir": "fwd", "seqs": 16, "toks": 7, "vocab": 97, "extra": 31, "x": "bf16"},
		# gradient of token log-probabilities over the text tower's vocabulary and context length
		{"name": "logprob_bwd_text", "op": "logprob", "dir": "bwd", "seqs": 64, "toks": 77, "vocab": 49408, "extra": 0, "x": "f16"},
		# a whole preference step of the label decoder: 4096 pairs of a right and a wrong label, loss and gradient
		{"name": "preference_step", "op": "preference", "seqs": 8192, "toks": 7, "vocab": 6912, "extra": 0, "x": "bf16", "kind": "sigmoid", "smoothing": 0.0, "weighted": True},
		# few pairs of long answers in single precision, an odd vocabulary
		{"name": "preference_long", "op": "preference", "seqs": 16, "toks": 333, "vocab": 10007, "extra": 0, "x": "f32", "kind": "sigmoid", "smoothing": 0.1, "weighted": False},
		# a whole policy step: 8192 sampled labels with one advantage each, clipped ratio and KL to the frozen decoder
		{"name": "policy_step", "op": "policy", "seqs": 8192, "toks": 7, "vocab": 6912, "extra": 0, "x": "bf16", "kl": 0.05, "per_seq": False},
		# six sampled labels over a vocabulary one short of a multiple, averaged label by label
		{"name": "policy_small", "op": "policy", "seqs": 6, "toks": 12, "vocab": 6911, "extra": 1, "x": "f32", "kl": 0.0, "per_seq": True},
	]


def _log_between(rng, lo, hi):
	return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
	op = rng.choice(["norm", "dropout", "logprob", "preference", "policy"])
	if op in ("norm", "dropout"):
		cols = _log_between(rng, 16, 16384)
		rows = _log_between(rng, 1, min(65792, 65792 * 1280 // cols))
		if rng.random() < 0.5 and cols > 64:
			cols -= cols % 64
		c = {"op": op, "dir": rng.choice(["fwd", "bwd"]), "rows": rows, "cols": cols, "resid": rng.random() < 0.5}
		if op == "norm":
			c["x"], c["y"] = rng.choice([("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
			c["beta"] = rng.random() < 0.5
			c["resid"] = c["resid"] and c["dir"] == "bwd"
		else:
			c["x"], c["y"] = rng.choice([("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
			c["p"] = rng.choice([0.1, round(rng.uniform(0.01, 0.9), 3)])
			c["resid"] = c["resid"] and c["dir"] == "fwd"
		return c
	room = 8192 * 7 * 6912
	x = rng.choice(["f32", "bf16", "f16"])
	vocab = _log_between(rng, 33, 131072)
	toks = _log_between(rng, 1, 512)
	seqs = 2 * _log_between(rng, 1, max(1, min(4096, room // (vocab * toks * (2 if x == "f32" else 1)) // 2)))
	c = {"op": op, "seqs": seqs, "toks": toks, "vocab": vocab, "extra": rng.choice([0, 0, (64 - vocab) % 64, 3]), "x": x}
	if op == "logprob":
		c["dir"] = rng.choice(["fwd", "bwd"])
	elif op == "preference":
		c["kind"] = rng.choice(["sigmoid", "sigmoid", "square"])
		c["smoothing"] = rng.choice([0.0, 0.1]) if c["kind"] == "sigmoid" else 0.0
		c["weighted"] = rng.random() < 0.5
	else:
		c["kl"] = rng.choice([0.0, 0.05])
		c["per_seq"] = rng.random() < 0.5
	return c


# ---- inputs --------------------------------------------------------------------------------------------------------------------

BETA, CLIP_LO, CLIP_HI = 0.1, 0.2, 0.28
SCALE = {"f32": 1.0, "bf16": 1.0, "f16": 16384.0}  # half-precision gradients are made under a loss scale, as any program does: they would leave the type's range


def _lengths(case, seed):
	"""Tokens of every sequence, from the seed alone: labels of one token up to the full length (work() asks for their sum with the seed that stands for all)."""
	return np.random.RandomState(seed % (1 << 31)).randint(1, case["toks"] + 1, case["seqs"])


def prepare(case, seed):
	g = torch.Generator(device="cuda").manual_seed(seed)
	dev = "cuda"

	def normal(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
		return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).mul_(scale).add_(shift).to(dtype)

	s = {"case": dict(case)}
	if case["op"] in ("norm", "dropout"):
		M, E, tx, ty = case["rows"], case["cols"], DTYPES[case["x"]], DTYPES[case["y"]]
		if case["op"] == "norm":
			s["x"] = normal(M, E, dtype=tx, scale=1.5, shift=0.2)
			s["gamma"], s["beta"] = normal(E, scale=0.2, shift=1.0), (normal(E, scale=0.2) if case["beta"] else None)
			s["mean"], s["rstd"] = torch.empty(M, device=dev), torch.empty(M, device=dev)
			if case["dir"] == "fwd":
				s["out"] = torch.empty(M, E, device=dev, dtype=ty)
			else:  # the statistics that the forward pass has kept
				x = s["x"].double()
				s["mean"].copy_(x.mean(1))
				s["rstd"].copy_((x.var(1, unbiased=False) + EPS).rsqrt())
				s["dy"] = normal(M, E, dtype=ty, scale=0.1)
				s["dx_in"] = normal(M, E, dtype=tx, scale=0.1) if case["resid"] else None
				s["dx"] = torch.empty(M, E, device=dev, dtype=tx)
				s["dgamma"], s["dbeta"] = torch.empty(E, device=dev), (torch.empty(E, device=dev) if case["beta"] else None)
		else:
			s["p"], s["seed"], s["site"] = case["p"], (seed * 0x9E3779B97F4A7C15 + 12345) & 0xFFFFFFFFFFFFFFFF, 7
			s["step"] = torch.full((), 1000 + seed % 1000, dtype=torch.int64, device=dev)
			a, b = (tx, ty) if case["dir"] == "fwd" else (ty, tx)
			s["in"], s["out"] = normal(M, E, dtype=a), torch.empty(M, E, device=dev, dtype=b)
			s["resid"] = normal(M, E, dtype=ty) if case["resid"] else None
		return s
	A, T, V, dt = case["seqs"], case["toks"], case["vocab"], DTYPES[case["x"]]
	R = A * T
	logits = torch.empty(R, V + case["extra"], device=dev, dtype=dt)
	for r0 in range(0, R, 8192):  # piece by piece: a step's logits in single precision need not exist at once
		logits[r0:r0 + 8192] = normal(min(8192, R - r0), V + case["extra"], scale=2.0)
	s["logits"] = logits[:, :V]
	s["target"] = torch.randint(0, V, (A, T), generator=g, device=dev)
	length = torch.from_numpy(_lengths(case, seed)).to(dev)
	s["pad"] = torch.arange(T, device=dev).unsqueeze(0) >= length.unsqueeze(1)
	s["target"].masked_fill_(s["pad"], 0)
	s["logp"], s["lse"] = torch.empty(A, T, device=dev), torch.empty(R, device=dev)
	if case["op"] == "logprob" and case["dir"] == "fwd":
		return s
	s["dlogits"] = torch.empty(R, V, device=dev, dtype=dt)
	logp, lse = torch.empty(R, device=dev), s["lse"]
	flat = s["target"].view(R, 1)
	for r0 in range(0, R, 8192):
		x = s["logits"][r0:r0 + 8192].float()
		lse[r0:r0 + 8192] = torch.logsumexp(x, 1)
		logp[r0:r0 + 8192] = x.gather(1, flat[r0:r0 + 8192]).squeeze(1) - lse[r0:r0 + 8192]
	logp = logp.view(A, T).masked_fill(s["pad"], 0.0)
	if case["op"] == "logprob":  # what a forward pass has kept, and the gradient that came down to the log-probabilities
		s["grad"] = normal(A, T, scale=SCALE[case["x"]] / R)
	elif case["op"] == "preference":  # the frozen decoder: the trained one has moved from it, towards the preferred half
		drift = torch.where(torch.arange(A, device=dev) < A // 2, -0.5, 0.5).unsqueeze(1)
		s["ref"] = (logp + drift + normal(A, T, scale=0.25)).masked_fill(s["pad"], 0.0)
		s["weight"] = torch.rand(A // 2, generator=g, device=dev).add_(0.5) if case["weighted"] else None
		s["stats"], s["z"] = torch.empty(3, device=dev), torch.empty(A // 2, device=dev)
	else:  # the policy that sampled, some updates ago: a third of the ratios lie outside the clip range, none within 1e-3 of its ends
		d = normal(A, T, scale=0.25)
		for end in (math.log(1 - CLIP_LO), math.log(1 + CLIP_HI)):
			near = (d - end).abs() < 1e-3
			d = torch.where(near, end + 2e-3 * torch.sign(d - end + 1e-9), d)
		s["old"] = (logp - d).masked_fill(s["pad"], 0.0)
		s["ref"] = (logp + normal(A, T, scale=0.3)).masked_fill(s["pad"], 0.0) if case["kl"] else None
		s["adv"] = normal(A)
		s["stats"] = torch.empty(4, device=dev)
	return s


# ---- the plain forms -----------------------------------------------------------------------------------------------------------

def _keep_plain(n, p, seed, site, step):
	"""Truth values of n elements: Philox4x32-10 with the key (seed) and the counter (element / 8, site, step), 16 bits an element, kept from round(65536 p) up."""
	mask = 0xFFFFFFFF
	block = torch.arange((n + 7) // 8, device="cuda", dtype=torch.int64)
	c0, c1, c2, c3 = block & mask, block >> 32, torch.full_like(block, site & mask), (step & mask).expand_as(block)
	k0, k1 = seed & mask, (seed >> 32) & mask
	for _ in range(10):
		a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
		c0, c1, c2, c3 = ((b >> 32) & mask) ^ c1 ^ k0, b & mask, ((a >> 32) & mask) ^ c3 ^ k1, a & mask
		k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
	words = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], 1).view(-1)[:n]
	return words >= int(p * 65536 + 0.5)


def _plain_norm(s, c):
	x = s["x"].float()
	if c["dir"] == "fwd":
		mean = x.sum(1, keepdim=True) / c["cols"]
		d = x - mean
		rstd = 1.0 / torch.sqrt((d * d).sum(1, keepdim=True) / c["cols"] + EPS)
		y = d * rstd * s["gamma"]
		if s["beta"] is not None:
			y = y + s["beta"]
		return {"y": y.to(DTYPES[c["y"]]), "mean": mean.squeeze(1), "rstd": rstd.squeeze(1)}
	dy, rstd = s["dy"].float(), s["rstd"].unsqueeze(1)
	xhat = (x - s["mean"].unsqueeze(1)) * rstd
	g = dy * s["gamma"]
	dx = rstd * (g - g.sum(1, keepdim=True) / c["cols"] - xhat * ((g * xhat).sum(1, keepdim=True) / c["cols"]))
	if s["dx_in"] is not None:
		dx = dx + s["dx_in"].float()
	out = {"dx": dx.to(DTYPES[c["x"]]), "dgamma": (dy * xhat).sum(0)}
	if s["dbeta"] is not None:
		out["dbeta"] = dy.sum(0)
	return out


def _plain_dropout(s, c):
	keep = _keep_plain(c["rows"] * c["cols"], s["p"], s["seed"], s["site"], s["step"]).view(c["rows"], c["cols"])
	y = torch.where(keep, s["in"].float() * (65536.0 / (65536 - int(s["p"] * 65536 + 0.5))), torch.zeros((), device="cuda"))
	if s["resid"] is not None:
		y = y + s["resid"].float()
	return {"y": y.to(s["out"].dtype)}


def _plain_logp(s):
	x = s["logits"].float()
	top = x.max(1, keepdim=True).values
	e = torch.exp(x - top)
	total = e.sum(1, keepdim=True, dtype=torch.float64)  # in 64 bits, and the log-probabilities with it: what the losses add up nearly cancels
	logp = ((x.gather(1, s["target"].view(-1, 1)) - top).double() - torch.log(total)).view(s["target"].shape).masked_fill(s["pad"], 0.0)
	return logp, e / total.float(), (top + torch.log(total)).float().squeeze(1)


def _plain_dlogits(s, p, grad):
	"""grad[A][T] (1[v = target] - p)"""
	g = grad.float().masked_fill(s["pad"], 0.0).view(-1, 1)
	return (-g * p).scatter_add_(1, s["target"].view(-1, 1), g).to(s["logits"].dtype)


def _plain_logprob(s, c):
	if c["dir"] == "fwd":
		logp, _, lse = _plain_logp(s)
		return {"logp": logp.float(), "lse": lse.masked_fill(s["pad"].view(-1), 0.0)}
	return {"dlogits": _plain_dlogits(s, torch.exp(s["logits"].float() - s["lse"].unsqueeze(1)), s["grad"])}


def _plain_preference(s, c):
	logp, p, _ = _plain_logp(s)
	n = c["seqs"] // 2
	ratio = (logp - s["ref"].double()).masked_fill(s["pad"], 0.0).sum(1)
	z = BETA * (ratio[:n] - ratio[n:])
	w = s["weight"].double() if s["weight"] is not None else torch.ones_like(z)
	if c["kind"] == "sigmoid":
		soft = torch.log(1.0 + torch.exp(-z.abs()))
		loss = (1 - c["smoothing"]) * (soft + torch.relu(-z)) + c["smoothing"] * (soft + torch.relu(z))
		dz = 1.0 / (1.0 + torch.exp(-z)) - (1 - c["smoothing"])
	else:
		u = z / BETA - 0.5 / BETA
		loss, dz = u * u, 2.0 * u / BETA
	dz = dz * w / w.sum() * BETA * SCALE[c["x"]]
	grad = torch.cat([dz, -dz]).unsqueeze(1).expand(-1, c["toks"])
	return {"stats": torch.stack([(w * loss).sum() / w.sum(), (w * z).sum() / w.sum(), w.sum()]).float(), "z": z.float(), "logp": logp.float(), "dlogits": _plain_dlogits(s, p, grad)}


def _plain_policy(s, c):
	logp, p, _ = _plain_logp(s)
	keep = ~s["pad"]
	lp, old, adv = logp, s["old"].double(), s["adv"].double().unsqueeze(1)
	r = torch.exp(lp - old)
	clipped = torch.clamp(r, 1 - CLIP_LO, 1 + CLIP_HI)
	whole = r * adv <= clipped * adv
	loss = -torch.where(whole, r * adv, clipped * adv)
	dlp = torch.where(whole, -r * adv, torch.zeros_like(r))
	kl = torch.zeros_like(r)
	if s["ref"] is not None:
		d = s["ref"].double() - lp
		kl = torch.exp(d) - d - 1.0
		loss, dlp = loss + c["kl"] * kl, dlp + c["kl"] * (1.0 - torch.exp(d))
	if c["per_seq"]:
		share = keep / keep.sum(1, keepdim=True).clamp(min=1) / keep.any(1).sum()
	else:
		share = keep / keep.sum()
	mean = lambda t: (torch.where(keep, t, torch.zeros_like(t)) * share).sum()  # noqa: E731
	stats = torch.stack([mean(loss), mean(kl), mean((~whole).double()), keep.sum().double()]).float()
	return {"stats": stats, "logp": logp.float(), "dlogits": _plain_dlogits(s, p, dlp * share * SCALE[c["x"]])}


def run(state):
	s, c = state, state["case"]
	if own:
		return _own(s, c)
	return {"norm": _plain_norm, "dropout": _plain_dropout, "logprob": _plain_logprob, "preference": _plain_preference, "policy": _plain_policy}[c["op"]](s, c)


def _own(s, c):
	from novic_amd import ops
	if c["op"] == "norm":
		if c["dir"] == "fwd":
			ops.layernorm_stats_fwd(s["x"], s["gamma"], s["beta"], s["out"], s["mean"], s["rstd"], eps=EPS)
			return {"y": s["out"], "mean": s["mean"], "rstd": s["rstd"]}
		ops.layernorm_stats_bwd(s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"], s["dx"], s["dgamma"], s["dbeta"], dx_in=s["dx_in"])
		return {"dx": s["dx"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]} if s["dbeta"] is not None else {"dx": s["dx"], "dgamma": s["dgamma"]}
	if c["op"] == "dropout":
		drop = ops.Dropout(s["p"], s["seed"], s["site"])
		if c["dir"] == "fwd":
			ops.dropout_fwd(s["in"], s["out"], drop, resid=s["resid"], step=s["step"])
		else:
			ops.dropout_bwd(s["in"], s["out"], drop, step=s["step"])
		return {"y": s["out"]}
	if c["op"] == "logprob":
		if c["dir"] == "fwd":
			ops.token_logprobs(s["logits"], s["target"], s["logp"], pad=s["pad"], lse=s["lse"])
			return {"logp": s["logp"], "lse": s["lse"]}
		ops.token_logprobs_bwd(s["logits"], s["target"], s["lse"], s["grad"], s["dlogits"], pad=s["pad"])
		return {"dlogits": s["dlogits"]}
	if c["op"] == "preference":
		ops.preference_loss(s["logits"], s["target"], s["ref"], s["stats"], beta=BETA, kind=c["kind"], smoothing=c["smoothing"], pad=s["pad"], weight=s["weight"],
		                    logp=s["logp"], margin=s["z"], dlogits=s["dlogits"], grad_scale=SCALE[c["x"]])
		return {"stats": s["stats"], "z": s["z"], "logp": s["logp"], "dlogits": s["dlogits"]}
	ops.policy_loss(s["logits"], s["target"], s["old"], s["adv"], s["stats"], clip=(CLIP_LO, CLIP_HI), ref=s["ref"], kl_coef=c["kl"], per_sequence=c["per_seq"], pad=s["pad"],
	                logp=s["logp"], dlogits=s["dlogits"], grad_scale=SCALE[c["x"]])
	return {"stats": s["stats"], "logp": s["logp"], "dlogits": s["dlogits"]}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------

def work(case):
	if case["op"] in ("norm", "dropout"):
		n, bx, by = case["rows"] * case["cols"], SIZE[case["x"]], SIZE[case["y"]]
		if case["op"] == "dropout":
			return {"bytes": n * (bx + by * (2 if case["resid"] else 1)), "flops": 2 * n}
		affine = 4 * case["cols"] * (2 if case["beta"] else 1)
		if case["dir"] == "fwd":
			return {"bytes": n * (bx + by) + 8 * case["rows"] + affine, "flops": 8 * n}
		return {"bytes": n * (by + bx * (3 if case["resid"] else 2)) + 8 * case["rows"] + 4 * case["cols"] + affine, "flops": 14 * n}
	rows, size = case["seqs"] * case["toks"], SIZE[case["x"]]
	counted = (case["seqs"] * (case["toks"] + 1)) // 2  # lengths are uniform in 1 .. toks: padded rows need not be read
	small = rows * (8 + 1 + 4)
	if case["op"] == "logprob" and case["dir"] == "fwd":
		return {"bytes": counted * case["vocab"] * size + small + 4 * rows, "flops": 4 * counted * case["vocab"]}
	return {"bytes": (counted + rows) * case["vocab"] * size + small + 8 * rows, "flops": 6 * counted * case["vocab"]}


# ---- the definitions in 64 bits, written apart ---------------------------------------------------------------------------------

def _exact_keep(n, p, seed, site, step):
	lo, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
	block = np.arange((n + 7) // 8, dtype=np.uint64)
	ctr = [block & lo, block >> s32, np.full_like(block, site), np.full_like(block, step & 0xFFFFFFFF)]
	key = [seed & 0xFFFFFFFF, seed >> 32]
	for r in range(10):
		kx, ky = np.uint64((key[0] + r * 0x9E3779B9) % (1 << 32)), np.uint64((key[1] + r * 0xBB67AE85) % (1 << 32))
		p0, p1 = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
		ctr = [(p1 >> s32) ^ ctr[1] ^ kx, p1 & lo, (p0 >> s32) ^ ctr[3] ^ ky, p0 & lo]
	u = np.stack(ctr, 1).astype("<u4").view("<u2").reshape(-1)[:n]
	return u >= math.floor(p * 65536 + 0.5)


def exact(case, seed):
	s = prepare(case, seed)
	wide = lambda t: None if t is None else t.detach().double()  # noqa: E731
	if case["op"] == "norm":
		x, gamma = wide(s["x"]), wide(s["gamma"])
		beta = wide(s["beta"]) if s["beta"] is not None else torch.zeros_like(gamma)
		if case["dir"] == "fwd":
			var, mu = torch.var_mean(x, 1, unbiased=False, keepdim=True)
			r = (var + EPS) ** -0.5
			return {"y": (x - mu) * r * gamma + beta, "mean": mu[:, 0], "rstd": r[:, 0]}
		# the gradient in terms of the kept statistics, which are inputs here
		dy, r = wide(s["dy"]), wide(s["rstd"])[:, None]
		n = (x - wide(s["mean"])[:, None]) * r
		up = dy * gamma
		dx = (up - up.mean(1, keepdim=True) - n * (up * n).mean(1, keepdim=True)) * r
		dx = dx if s["dx_in"] is None else dx + wide(s["dx_in"])
		out = {"dx": dx, "dgamma": torch.einsum("me,me->e", dy, n)}
		return out if s["dbeta"] is None else {**out, "dbeta": dy.sum(0)}
	if case["op"] == "dropout":
		keep = torch.from_numpy(_exact_keep(case["rows"] * case["cols"], case["p"], s["seed"], s["site"], int(s["step"]))).cuda().view(case["rows"], case["cols"])
		thr = math.floor(case["p"] * 65536 + 0.5)
		y = wide(s["in"]) * keep * (1.0 / (1.0 - thr / 65536.0))
		return {"y": y if s["resid"] is None else y + wide(s["resid"])}
	A, T, V = case["seqs"], case["toks"], case["vocab"]
	x = wide(s["logits"])
	some = (~s["pad"]).double()
	if case["op"] == "logprob" and case["dir"] == "bwd":  # lse is an input here
		x.sub_(s["lse"].double()[:, None]).exp_().neg_()
		x[torch.arange(A * T, device="cuda"), s["target"].view(-1)] += 1.0
		return {"dlogits": x.mul_((s["grad"].double() * some).view(-1, 1))}
	lse = torch.logsumexp(x, 1)
	lp = ((x[torch.arange(A * T, device="cuda"), s["target"].view(-1)] - lse).view(A, T) * some).requires_grad_()
	if case["op"] == "logprob":
		return {"logp": lp.detach(), "lse": lse * some.view(-1)}
	if case["op"] == "preference":
		gain = ((lp - wide(s["ref"])) * some).sum(1).view(2, A // 2)
		z = BETA * (gain[0] - gain[1])
		w = torch.ones_like(z) if s["weight"] is None else wide(s["weight"])
		if case["kind"] == "sigmoid":
			e = case["smoothing"]
			each = -(1 - e) * torch.nn.functional.logsigmoid(z) - e * torch.nn.functional.logsigmoid(-z)
		else:
			each = (gain[0] - gain[1] - 1 / (2 * BETA)) ** 2
		loss = (each * w).sum() / w.sum()
		out = {"stats": torch.stack([loss.detach(), ((z * w).sum() / w.sum()).detach(), w.sum()]), "z": z.detach()}
	else:
		count = some.sum()
		share = some / some.sum(1, keepdim=True) / A if case["per_seq"] else some / count
		r, a = (lp - wide(s["old"])).exp(), wide(s["adv"])[:, None]
		held = r.clamp(1 - CLIP_LO, 1 + CLIP_HI)
		each = -torch.minimum(r * a, held * a)
		kl = torch.zeros_like(r)
		if s["ref"] is not None:
			kl = (wide(s["ref"]) - lp).exp() - 1 - (wide(s["ref"]) - lp)
			each = each + case["kl"] * kl
		loss = (each * share).sum()
		cut = (((r > 1 + CLIP_HI) & (a > 0)) | ((r < 1 - CLIP_LO) & (a < 0))).double()
		out = {"stats": torch.stack([loss.detach(), (kl * share).sum().detach(), (cut * share).sum().detach(), count])}
	(dlp,) = torch.autograd.grad(loss * SCALE[case["x"]], lp)
	x.sub_(lse[:, None]).exp_().neg_()
	x[torch.arange(A * T, device="cuda"), s["target"].view(-1)] += 1.0
	return {**out, "logp": lp.detach(), "dlogits": x.mul_((dlp * some).view(-1, 1))}
