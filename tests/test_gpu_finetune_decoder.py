"""Preference and policy steps of the label decoder (PrefixedIterDecoder.token_logprobs, forward_backward_preference, forward_backward_policy) against the CPU oracle with autograd.

Tolerances are those of the decoder's other parity tests, for the same chain of bf16 products: gradients within 6e-2 relative 2-norm per tensor; a log-probability is off by at most
what its logit and its row's log-sum-exp are, 3e-2 of the largest logit each.  The losses' inputs are made from the oracle's log-probabilities, with ratios away from the clip range's ends by more
than that."""
import pytest
import torch

from helpers import make_decoder, synth_batch, to_dev
from novic_amd import train as T
from oracle import decoder_oracle as O

pytestmark = pytest.mark.gpu

SPECS = {"small": dict(embed_dim=32, vocab_size=53, token_length=6, hidden_dim=64, feedfwd_dim=16, num_layers=2, num_heads=4),
         "released_layer": dict(embed_dim=512, vocab_size=307, token_length=8, num_layers=1)}


def rel_l2(a, b):
	return float((a.float() - b.float()).norm() / (b.float().norm() + 1e-12))


def setup(name, B, M, seed=17):
	spec = O.DecoderSpec(**SPECS[name])
	model, sd = make_decoder(spec, seed=seed, device="cuda")
	embed, target, pad, _ = synth_batch(spec, B, seed=5, M=M)
	return spec, model, sd, embed, target, pad


def oracle_logprobs(sd, spec, embed, target, pad):
	"""[A][C] log-probabilities with their graph, zeros at padded positions."""
	logits = O.forward(sd, spec, embed, target, pad, None, False, False, False)[0]
	logp = torch.log_softmax(logits, -1).gather(-1, target.long().clamp(min=0).unsqueeze(-1)).squeeze(-1)
	return torch.where(pad, torch.zeros(()), logp), float(logits.detach().abs().max())


@pytest.mark.parametrize("name", SPECS)
@pytest.mark.parametrize("kind,smoothing,weighted", [("sigmoid", 0.1, True), ("square", 0.0, False)])
def test_preference_step(name, kind, smoothing, weighted):
	spec, model, sd, embed, target, pad = setup(name, 7, 2)
	model.eval()  # dropout off, exact comparison
	sdg = {k: (v.clone().requires_grad_(True) if k != "causality_mask" else v) for k, v in sd.items()}
	both = torch.cat([embed, embed])
	t2, p2 = target.transpose(0, 1).contiguous(), pad.transpose(0, 1).contiguous()  # [2][B][C]
	logp, top = oracle_logprobs(sdg, spec, both, t2.reshape(-1, t2.shape[-1]), p2.reshape(-1, t2.shape[-1]))
	g = torch.Generator().manual_seed(1)
	ref = torch.where(p2.reshape(logp.shape), torch.zeros(()), logp.detach() + 0.3 * torch.randn(logp.shape, generator=g))
	w = torch.rand(7, generator=g) + 0.5 if weighted else torch.ones(7)
	beta = 0.5
	u = (logp - ref).sum(1)
	z = beta * (u[:7] - u[7:])
	each = -(1 - smoothing) * torch.nn.functional.logsigmoid(z) - smoothing * torch.nn.functional.logsigmoid(-z) if kind == "sigmoid" else ((z - 0.5) / beta) ** 2
	loss = (w * each).sum() / w.sum()
	(3.0 * loss).backward()
	args = to_dev(embed, t2, p2, ref.view(t2.shape))
	call = lambda: model.forward_backward_preference(*args, beta=beta, kind=kind, smoothing=smoothing, weight=w.cuda() if weighted else None, loss_scale=3.0)  # noqa: E731
	stats, margin, got = call()
	assert got.shape == t2.shape and not got.cpu()[p2].any()
	off = 2 * 3e-2 * max(1.0, top)
	assert float((got.cpu().view(logp.shape) - logp.detach()).abs().max()) <= off
	assert torch.equal(model.token_logprobs(*args[:3]), got)  # dropout off: the frozen decoder's are the same numbers
	assert abs(float(stats[0]) - float(loss.detach())) <= 6e-2 * max(1.0, float(loss.detach())) and abs(float(stats[2]) - float(w.sum())) < 1e-4
	assert float((margin.cpu() - z.detach()).abs().max()) <= beta * 2 * t2.shape[-1] * off
	for k, p in model.named_parameters():
		assert rel_l2(p.grad.cpu(), sdg[k].grad) <= 6e-2, k
	call()  # accumulates
	for k, p in model.named_parameters():
		assert rel_l2(p.grad.cpu(), 2 * sdg[k].grad) <= 6e-2, k


@pytest.mark.parametrize("name", SPECS)
@pytest.mark.parametrize("kl,per_seq,adv_dim", [(0.0, False, 1), (0.2, True, 2)])
def test_policy_step(name, kl, per_seq, adv_dim):
	spec, model, sd, embed, target, pad = setup(name, 9, None)
	model.eval()
	sdg = {k: (v.clone().requires_grad_(True) if k != "causality_mask" else v) for k, v in sd.items()}
	logp, top = oracle_logprobs(sdg, spec, embed, target, pad)
	g = torch.Generator().manual_seed(2)
	d = torch.where(torch.rand(logp.shape, generator=g) < 0.3, 0.9, 0.0) * torch.where(torch.rand(logp.shape, generator=g) < 0.5, -1.0, 1.0)
	old = torch.where(pad, torch.zeros(()), logp.detach() - d)
	ref = torch.where(pad, torch.zeros(()), logp.detach() + 0.4 * torch.randn(logp.shape, generator=g))
	adv = torch.randn(9, generator=g) if adv_dim == 1 else torch.randn(logp.shape, generator=g)
	q, a = (logp - old).exp(), adv[:, None].expand_as(logp) if adv_dim == 1 else adv
	each = -torch.minimum(q * a, q.clamp(0.6, 1.6) * a) + kl * (torch.expm1(ref - logp) - (ref - logp))
	keep = ~pad
	share = keep / keep.sum(1, keepdim=True) / 9 if per_seq else keep / keep.sum()
	loss = (each * share).sum()
	loss.backward()
	stats, got = model.forward_backward_policy(*to_dev(embed, target, pad, old, adv), clip=(0.4, 0.6), ref_logprobs=ref.cuda() if kl else None, kl_coef=kl, per_sequence=per_seq)
	off = 2 * 3e-2 * max(1.0, top)
	assert float((got.cpu() - logp.detach()).abs().max()) <= off
	assert abs(float(stats[0]) - float(loss.detach())) <= 6e-2 * max(1.0, abs(float(loss.detach()))) and float(stats[3]) == float(keep.sum())
	for k, p in model.named_parameters():
		assert rel_l2(p.grad.cpu(), sdg[k].grad) <= 6e-2, k


def test_steps_with_dropout_and_the_optimizer():
	"""Preference and policy steps in training mode, through the fused optimizer, from a frozen twin's log-probabilities: everything stays finite."""
	spec, model, sd, embed, target, pad = setup("released_layer", 16, 2)
	frozen, _ = make_decoder(spec, seed=17, device="cuda")
	model, _ = make_decoder(spec, seed=17, dropout=0.1, device="cuda")
	model.train()
	opt = T.FusedAdamW(model, lr=1e-3)
	args = to_dev(embed, target.transpose(0, 1).contiguous(), pad.transpose(0, 1).contiguous())
	ref = frozen.token_logprobs(*args)
	assert torch.equal(ref, frozen.token_logprobs(*args))
	for _ in range(3):
		opt.zero_grad()
		stats, margin, logp = model.forward_backward_preference(*args, ref, beta=0.1)
		norm = opt.step()
		assert torch.isfinite(stats).all() and torch.isfinite(margin).all() and torch.isfinite(norm).all() and float(norm) > 0
	one = (args[0], args[1][0].contiguous(), args[2][0].contiguous())
	old = model.token_logprobs(*one)
	opt.zero_grad()
	stats, logp = model.forward_backward_policy(*one, old, torch.ones(16, device="cuda"), ref_logprobs=ref[0].contiguous(), kl_coef=0.05)
	norm = opt.step()
	assert torch.isfinite(stats).all() and float(norm) > 0


def test_refusals():
	spec, model, sd, embed, target, pad = setup("small", 4, 2)
	e, t, p = to_dev(embed, target, pad)
	f = torch.zeros(target.shape, device="cuda")
	with pytest.raises(ValueError):
		model.forward_backward_preference(e, t, p, f)           # [B][2][C]
	with pytest.raises(ValueError):
		model.forward_backward_preference(e, t[:, 0], p[:, 0], f[:, 0])
	with pytest.raises(ValueError):
		model.forward_backward_policy(e, t, p, f, f)
	t2, p2, f2 = (x.transpose(0, 1).contiguous() for x in (t, p, f))
	with pytest.raises(ValueError):
		model.forward_backward_preference(e, t2, p2, f2, kind="other")
	with pytest.raises(ValueError):
		model.forward_backward_preference(e, t2, p2, f2[:, :2])
	with pytest.raises(ValueError):
		model.forward_backward_preference(e, t2, p2, f)         # as many numbers in another order
	with pytest.raises(ValueError):
		model.forward_backward_preference(e[:0], t2[:, :0], p2[:, :0], f2[:, :0])
	assert model.token_logprobs(e[:0], t2[:, :0], p2[:, :0]).shape == (2, 0, t2.shape[2])
	with pytest.raises(AssertionError):
		model.forward_backward_preference(e[:3], t2, p2, f2)


def test_strided_targets_and_end_losses():
	"""Targets and padding of any strides give the same numbers, and tokens the cross entropy counts behind a label's end (num_end_loss) are no part of its log-probability."""
	spec, model, sd, embed, target, pad = setup("small", 5, None)
	e, t, p = to_dev(embed, target, pad)
	want = model.token_logprobs(e, t, p)
	wide_t, wide_p = t.new_zeros(t.shape[1], t.shape[0]), p.new_zeros(5, 2 * p.shape[1])
	wide_t.copy_(t.t())
	wide_p[:, ::2] = p
	assert torch.equal(model.token_logprobs(e, wide_t.t(), wide_p[:, ::2]), want)
	model.num_end_loss = 3
	assert torch.equal(model.token_logprobs(e, t, p).masked_fill(p, 0), want)
