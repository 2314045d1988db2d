"""The operators of decoder fine-tuning (novic_amd/ops.py: layernorm_stats_*, dropout_*, token_logprobs*, preference_loss, policy_loss) refuse what they cannot do, before anything is
launched.  The C ABI is called with addresses that no check may follow: a call that got past its checks would fail to launch here, with another message."""
import ctypes
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from novic_amd import _lib, ops

MiB = 1 << 20
P = 4096  # an address


def at(k):
	return (k + 1) << 30


@pytest.fixture(scope="module", autouse=True)
def library():
	if not os.path.exists(_lib.LIB_PATH):
		_lib.build()
	return _lib.lib()


def refused(name, args, why):
	rc = ops._entry(name)(*args, 0)
	assert rc == -22, f"{name} accepted {args}"
	assert why in _lib.lib().novic_last_error().decode(), _lib.lib().novic_last_error()


def change(args, **at):
	args = list(args)
	for k, v in at.items():
		args[int(k[1:])] = v
	return args


LN_FWD = [at(0), 0, 64, P, 0, at(1), 1, 64, 0, 0, 4, 64, 1e-5]
LN_BWD = [at(0), 1, 64, at(1), 0, 64, P, at(2), at(3), 0, 0, at(4), 64, at(5), at(6), 0, 400, 64, at(7), 1 << 20]
DROP = [at(0), 0, 64, 0, 0, at(1), 0, 64, 4, 64, 0.1, 1, 2, 0]
ROWS = [at(0), 1, 64, P, 8, 7, at(1), 7, 4, 7, 64]
LOGP = ROWS + [at(2), 7, 0]
LOGP_BWD = ROWS + [at(2), at(3), 7, 1, at(4), 64]
PREF = ROWS + [at(2), 7, 0, 0, 0.1, 0.0, 1.0, 0, 7, 0, 0, 64, at(3), at(4), 1 << 20]
POLICY = ROWS + [at(2), 7, at(3), 1, 0, 0, 7, 0.2, 0.2, 0.0, 0, 1.0, 0, 7, 0, 64, at(4), at(5), 1 << 20]


@pytest.mark.parametrize("change_,why", [(dict(_11=0), "E <= 16384"), (dict(_11=16385), "E <= 16384"), (dict(_2=63), "leading dimensions"), (dict(_7=8), "leading dimensions"),
                                         (dict(_10=-1), "rows >= 0"), (dict(_1=1, _6=0), "x's type"), (dict(_1=3), "x's type"), (dict(_0=0), "null"), (dict(_3=0), "null"), (dict(_5=0), "null")])
def test_layernorm_forward(change_, why):
	refused("novic_layernorm_stats_fwd", change(LN_FWD, **change_), why)


@pytest.mark.parametrize("change_,why", [(dict(_17=16385), "E <= 16384"), (dict(_2=63), "leading"), (dict(_5=63), "leading"), (dict(_12=63), "leading"), (dict(_9=at(8), _10=63), "leading"),
                                         (dict(_4=1, _1=2), "x's type"), (dict(_7=0), "null"), (dict(_8=0), "null"), (dict(_18=0), "workspace"), (dict(_19=64), "workspace")])
def test_layernorm_backward(change_, why):
	refused("novic_layernorm_stats_bwd", change(LN_BWD, **change_), why)


@pytest.mark.parametrize("change_,why", [(dict(_10=-0.1), "p <= 1"), (dict(_10=1.5), "p <= 1"), (dict(_10=float("nan")), "p <= 1"), (dict(_2=63), "leading"), (dict(_7=63), "leading"),
                                         (dict(_3=at(8), _4=63), "leading"), (dict(_1=1, _6=2), "types"), (dict(_1=-1), "type"), (dict(_0=0), "null"), (dict(_8=-1), "rows"),
                                         (dict(_8=1 << 40, _9=1 << 30, _2=1 << 30, _7=1 << 30), "too many")])
def test_dropout(change_, why):
	refused("novic_dropout", change(DROP, **change_), why)


SHARED = [(dict(_1=3), "fp32, bf16 or fp16"), (dict(_4=2), "tok_bytes"), (dict(_10=0), "V <= 2^28"), (dict(_10=(1 << 28) + 1, _2=1 << 29), "V <= 2^28"), (dict(_8=-4), "A, T >= 0"), (dict(_2=63), ">= V"), (dict(_5=6), "target and pad"), (dict(_7=6), "target and pad"),
          (dict(_0=0), "null"), (dict(_3=0), "null"), (dict(_8=1 << 30, _9=8, _5=8, _7=8), "2^31")]


@pytest.mark.parametrize("change_,why", SHARED)
@pytest.mark.parametrize("name", ["novic_token_logprobs", "novic_token_logprobs_bwd", "novic_preference_loss", "novic_policy_loss"])
def test_token_rows(name, change_, why):
	args = {"novic_token_logprobs": LOGP, "novic_token_logprobs_bwd": LOGP_BWD, "novic_preference_loss": PREF, "novic_policy_loss": POLICY}[name]
	if name == "novic_preference_loss" and change_.get("_8") is not None:
		change_ = dict(change_, _8=change_["_8"] // 2)
		why = "at least one" if change_["_8"] < 0 else why
	if name == "novic_policy_loss" and change_.get("_8", 1) < 0:
		why = "at least one"
	refused(name, change(args, **change_), why)


@pytest.mark.parametrize("change_,why", [(dict(_14=3), "kind"), (dict(_15=0.0), "beta"), (dict(_15=float("nan")), "beta"), (dict(_16=0.5), "smoothing"), (dict(_16=-0.1), "smoothing"),
                                         (dict(_14=1, _16=0.1), "smoothing"), (dict(_11=0), "ref"), (dict(_12=6), "ref"), (dict(_18=at(8), _19=6), "ref"), (dict(_23=0), "stats"), (dict(_24=0), "workspace"),
                                         (dict(_25=16), "workspace"), (dict(_8=0), "at least one"), (dict(_9=0), "at least one"), (dict(_21=at(8), _22=63), ">= V")])
def test_preference(change_, why):
	refused("novic_preference_loss", change(PREF, **change_), why)


@pytest.mark.parametrize("change_,why", [(dict(_18=-0.1), "clip"), (dict(_18=1.1), "clip"), (dict(_19=-0.1), "clip"), (dict(_20=-1.0), "kl_coef"), (dict(_20=float("nan")), "kl_coef"), (dict(_11=0), "old"),
                                         (dict(_13=0), "old"), (dict(_12=6), "old"), (dict(_16=at(8), _17=6), "old"), (dict(_27=0), "old"), (dict(_28=0), "workspace"), (dict(_29=8), "workspace"),
                                         (dict(_8=0), "at least one"), (dict(_9=0), "at least one")])
def test_policy(change_, why):
	refused("novic_policy_loss", change(POLICY, **change_), why)


def test_nothing_to_do_is_no_error():
	assert ops._entry("novic_layernorm_stats_fwd")(*change(LN_FWD, _10=0, _0=0), 0) == 0
	assert ops._entry("novic_dropout")(*change(DROP, _8=0, _0=0), 0) == 0
	assert ops._entry("novic_token_logprobs")(*change(LOGP, _8=0, _0=0), 0) == 0
	assert ops._entry("novic_token_logprobs_bwd")(*change(LOGP_BWD, _9=0, _0=0), 0) == 0
	assert _lib.lib().novic_layernorm_stats_bwd_ws(0, 64, 0, 0) == 0


def test_workspaces_grow_with_the_problem():
	lib = _lib.lib()
	for f in (lib.novic_preference_loss_ws, lib.novic_policy_loss_ws, lib.novic_layernorm_stats_bwd_ws):
		f.restype = ctypes.c_uint64
	assert lib.novic_preference_loss_ws(8, 7) >= 8 * 7 * 2 * 16 and lib.novic_preference_loss_ws(1 << 24, 64) > 1 << 32
	assert lib.novic_policy_loss_ws(8, 7) >= 8 * 7 * 12 and lib.novic_policy_loss_ws(1 << 24, 64) > 1 << 32
	assert lib.novic_layernorm_stats_bwd_ws(1 << 20, 16384, 1, 1) >= 2 * 16384 * 4


def test_cpu_tensors_are_refused():
	f, i = torch.zeros(4, 8), torch.zeros(2, 2, dtype=torch.int64)
	e, s = torch.zeros(8), torch.zeros(4)
	for call in (lambda: ops.layernorm_stats_fwd(f, e, None, f), lambda: ops.layernorm_stats_bwd(f, f, e, s, s, f), lambda: ops.dropout_fwd(f, f, ops.NO_DROPOUT),
	             lambda: ops.dropout_bwd(f, f, ops.NO_DROPOUT), lambda: ops.token_logprobs(f, i, f), lambda: ops.token_logprobs_bwd(f, i, s, f, f),
	             lambda: ops.preference_loss(f, i, f, s, beta=0.1), lambda: ops.policy_loss(f, i, f, s, s)):
		with pytest.raises(_lib.NovicHipError):
			call()
	with pytest.raises(TypeError):
		ops.layernorm_stats_fwd(None, e, None, f)


@pytest.mark.parametrize("name,args", [
	("novic_layernorm_stats_fwd", change(LN_FWD, _0=MiB, _5=MiB)),                      # y (bf16) on x (fp32)
	("novic_layernorm_stats_fwd", change(LN_FWD, _0=MiB, _5=MiB + 256, _6=0)),          # y one row into x
	("novic_layernorm_stats_fwd", change(LN_FWD, _0=MiB, _5=2 * MiB, _8=3 * MiB, _9=3 * MiB + 4)),  # mean on rstd
	("novic_layernorm_stats_bwd", change(LN_BWD, _9=0, _13=8 * MiB, _14=8 * MiB)),  # dgamma is dbeta
	("novic_layernorm_stats_bwd", change(LN_BWD, _9=0, _13=P, _14=0)),   # dgamma is gamma
	("novic_layernorm_stats_bwd", change(LN_BWD, _11=at(1) + 4, _13=0, _14=0)),
	("novic_dropout", change(DROP, _0=MiB, _5=MiB + 4)), ("novic_dropout", change(DROP, _0=MiB, _5=2 * MiB, _3=2 * MiB + 256, _4=64)), ("novic_dropout", change(DROP, _0=MiB, _5=2 * MiB, _13=2 * MiB + 8)),
	("novic_token_logprobs", change(LOGP, _0=MiB, _11=MiB + 128)), ("novic_token_logprobs", change(LOGP, _0=MiB, _3=P, _11=P + 32)),
	("novic_token_logprobs_bwd", change(LOGP_BWD, _0=MiB, _15=MiB + 2)), ("novic_token_logprobs_bwd", change(LOGP_BWD, _0=MiB, _11=3 * MiB, _12=3 * MiB, _15=3 * MiB)),
	("novic_preference_loss", change(PREF, _0=MiB, _8=2, _18=5 * MiB, _11=5 * MiB, _24=9 * MiB)),   # logp is ref
	("novic_preference_loss", change(PREF, _0=MiB, _8=2, _11=5 * MiB, _23=9 * MiB, _24=9 * MiB)),   # stats in the workspace
	("novic_policy_loss", change(POLICY, _0=MiB, _11=5 * MiB, _23=5 * MiB, _27=7 * MiB, _28=9 * MiB)),  # logp is old
	("novic_policy_loss", change(POLICY, _0=MiB, _11=5 * MiB, _25=MiB + 128, _27=7 * MiB, _28=9 * MiB)),
])
def test_overlaps(name, args):
	refused(name, args, "overlaps")


def test_overlaps_are_told_from_windows():
	"""Column windows of one buffer, and an output that is an input, pass this check: the next one, a null pointer or a small workspace put there, is what refuses the call."""
	refused("novic_layernorm_stats_bwd", change(LN_BWD, _1=0, _0=MiB, _2=256, _3=MiB + 256, _5=256, _11=MiB + 512, _12=256, _9=MiB + 768, _10=256, _13=8 * MiB, _14=0, _18=0), "workspace")
	refused("novic_layernorm_stats_bwd", change(LN_BWD, _1=0, _0=MiB, _2=64, _3=MiB, _5=64, _11=MiB, _12=64, _13=8 * MiB, _14=0, _18=0), "workspace")
	refused("novic_layernorm_stats_bwd", change(LN_BWD, _1=0, _0=MiB, _2=256, _3=MiB + 252, _5=256, _11=MiB + 512, _12=256, _13=8 * MiB, _14=0, _18=0), "workspace")  # (two inputs may overlap)
	refused("novic_layernorm_stats_bwd", change(LN_BWD, _1=0, _0=MiB, _2=256, _3=MiB + 256, _5=256, _11=MiB + 508, _12=256, _13=8 * MiB, _14=0, _18=0), "overlaps")
