"""A loss of PrefixedIterDecoder.forward() whose backward() is still to come, while the same decoder is asked for something else."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from helpers import make_decoder, synth_batch, to_dev
from oracle import decoder_oracle as O

pytestmark = pytest.mark.gpu
SPEC = O.DecoderSpec(embed_dim=32, vocab_size=53, token_length=6, hidden_dim=64, feedfwd_dim=16, num_layers=2, num_heads=4)


@pytest.fixture
def pending():
	"""(model in eval mode, a forward() of eight labels, its undisturbed gradients, the inputs of other calls)"""
	model, _ = make_decoder(SPEC, seed=17, device="cuda")
	model.eval()
	embed, target, pad, weight = to_dev(*synth_batch(SPEC, 8, seed=5))
	forward = lambda: model(embed, target, pad, weight, True, False, False, None)[2]  # noqa: E731
	grads = torch.autograd.grad(forward(), list(model.parameters()))
	other = to_dev(*synth_batch(SPEC, 8, seed=6))
	return model, forward, grads, other


@pytest.mark.parametrize("rows", [8, 3])
def test_log_probabilities_between_a_loss_and_its_gradient(pending, rows):
	"""token_logprobs has a workspace of its own: the waiting gradients are what they were, with labels of the same shape and with fewer of them."""
	model, forward, grads, (embed, target, pad, _) = pending
	want = model.token_logprobs(embed[:rows], target[:rows], pad[:rows])
	loss = forward()
	got = model.token_logprobs(embed[:rows], target[:rows], pad[:rows])
	assert torch.equal(got, want)
	# (looked at on the host before anything is launched: buffers of another call's size would be read and written past their ends)
	assert model._ws.bufs["fwd:logits"].shape[0] == 8 * target.shape[1] and model._ws.bufs["fwd:key_pad"].shape[0] == 8
	for (k, _), a, b in zip(model.named_parameters(), torch.autograd.grad(loss, list(model.parameters())), grads):
		# float atomics of the weight gradients: at most 64 rows' terms in another order, 64 * 2^-24 of their absolute sum, allowed to be 64 times the largest gradient
		assert float((a - b).abs().max()) <= 2.0 ** -12 * float(b.abs().max()), k


@pytest.mark.parametrize("rows", [8, 3])
def test_a_forward_without_gradients_ends_the_waiting_one(pending, rows):
	"""forward() has one workspace: another pass through it, without gradients too, writes over the activations, and the gradient that still waits for them is refused."""
	model, forward, grads, (embed, target, pad, _) = pending
	loss = forward()
	with torch.no_grad():
		model(embed[:rows], target[:rows], pad[:rows], None, True, False, False, None)
	with pytest.raises(RuntimeError, match="before the next forward"):
		loss.backward()
	again = torch.autograd.grad(forward(), list(model.parameters()))  # and the next pair is whole
	for (k, _), a, b in zip(model.named_parameters(), again, grads):
		assert float((a - b).abs().max()) <= 2.0 ** -12 * float(b.abs().max()), k
