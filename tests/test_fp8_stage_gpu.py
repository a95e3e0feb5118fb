"""Layers in 8 bits as stages and users' programs call them: several outputs, many micro-batches, layers used twice, outputs written in place.
Tolerances are those of test_fp8_layers_gpu.py."""

import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from tests.test_fp8_layers_gpu import E4M3, E5M2, make, moved, near, rnd

pytestmark = pytest.mark.gpu


def gen(seed):
	return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------------------------------------ several outputs
class _Cut(nn.Module):
	"""A stage that ends behind a ``NormLinear8``: its outputs are that layer's, and the layers before lie upstream of both."""

	def __init__(self, d=136, n=264):
		from elf_amd.models import Linear8, NormLinear8

		super().__init__()
		self.first, self.second = Linear8(d, d), NormLinear8(d, n)

	def forward(self, a):
		return self.second(self.first(a), a)


class _Both(nn.Module):
	"""Two outputs of one product."""

	def __init__(self, d=136, n=264):
		from elf_amd.models import Linear8, NormLinear8

		super().__init__()
		self.first, self.second = NormLinear8(d, d, bias=False), Linear8(d, n, grad_dtype=E5M2)

	def forward(self, a):
		h, y = self.first(a)
		z = self.second(h + y)
		return z, torch.tanh(z)


def _stage(kind, variant, T=70, n_mb=2):
	from elf_amd.execution import AutogradStageBlock
	from elf_amd.partitioners.utils import Signature
	from elf_amd.scheduling import OpOptions

	torch.manual_seed(21)
	model = kind().to(torch.bfloat16)
	ref = copy.deepcopy(model).float().cuda()
	blk = AutogradStageBlock(model, 1, [0, 1, 2], Signature(["a"], ["u", "v"], [0], [[2], [2]]))
	g = gen(22)
	data = [rnd(g, T, 136) for _ in range(n_mb)]
	blk.zero_grad()
	outs, dxs, dys = [], [], []
	for m in range(n_mb):
		blk.input_variables[0].set(blk.input_variables[0].to_process, m, (None, data[m].clone()))
		blk.forward(m, **({OpOptions.REMAT_STRATEGY: (lambda name, module: name == variant[6:])} if variant.startswith("remat_") else {}))
	for m in range(n_mb):
		dys.append([])
		for targets in blk.output_variables:
			y = targets[0].get(targets[0].to_send, m)
			outs.append(y)
			dys[-1].append(rnd(g, *y.shape, by=0.1))
			targets[0].set(targets[0].to_process, m, (None, dys[-1][-1]))
		if variant == "activations_bwd":
			blk.backward_inputs(m, **{OpOptions.RECOMPUTE_ACTIVATIONS: True})
			blk.recompute_forward(m)
		elif variant == "full_bwd":
			blk.backward_inputs(m, **{OpOptions.RECOMPUTE_ACTIVATIONS: True, OpOptions.RECOMPUTE_GRADIENTS: True})
			assert all(l.ctx["input"][m] is None and l.ctx["grad_output"][m] is None for l in blk._layers_dw())
			blk.recompute_forward(m, **{OpOptions.SAVE: True})
			blk.recompute_backward_inputs(m)
		else:
			blk.backward_inputs(m)
		dxs.append(blk.input_variables[0].get(blk.input_variables[0].to_send, m))
		blk.backward_params(m)
		assert all(l.ctx["input"][m] is None and l.ctx["grad_output"][m] is None for l in blk._layers_dw())
	params = {name: (p.main_grad if getattr(p, "main_grad", None) is not None else p.grad) for name, p in blk.model.named_parameters()}
	return ref, data, dys, outs, dxs, params


@pytest.mark.parametrize("kind", [_Cut, _Both])
def test_stage_whose_outputs_share_a_product(kind):
	ref, data, dys, outs, dxs, params = _stage(kind, "plain")
	want = []
	for a, gr, dx in zip(data, dys, dxs):
		a = a.float().requires_grad_(True)
		ys = ref(a)
		torch.autograd.backward(ys, [t.float() for t in gr])
		want += [y.detach() for y in ys]
		near(dx, a.grad, 0.15, "input gradient")
	for got, w in zip(outs, want):
		near(got, w, 0.15, "output")
	for name, p in ref.named_parameters():
		near(params[name], p.grad, 0.15, name)


@pytest.mark.parametrize("variant", ["remat_first", "remat_second", "activations_bwd", "full_bwd"])
@pytest.mark.parametrize("kind", [_Cut, _Both])
def test_variants_of_a_stage_whose_outputs_share_a_product(kind, variant):
	_, _, _, outs, dxs, params = _stage(kind, "plain")
	_, _, _, outs2, dxs2, params2 = _stage(kind, variant)
	for a, b in zip(outs + dxs, outs2 + dxs2):
		assert torch.equal(a, b)
	for name in params:
		assert torch.equal(params[name], params2[name]), name


def test_several_backward_calls_through_one_use():
	"""Output gradients that come one after the other are kept one by one, on the host too, and W adds the product of each."""
	from elf_amd import kernels as K
	from elf_amd.models import Linear8

	g = gen(23)
	layer = make(Linear8, 200, 72, True, E4M3, g)
	x = rnd(g, 50, 200).requires_grad_(True)
	dys = [rnd(g, 50, 72, by=0.1) for _ in range(3)]
	y = layer(x)
	for dy in dys:
		y.backward(dy, retain_graph=True)
	moved(layer, 0)
	layer.offload_last(0)
	torch.cuda.synchronize()
	layer.offload_last(0, to="cuda")
	layer.backward(0)
	acc, bias = torch.zeros(72, 200, device="cuda"), torch.zeros(72, device="cuda")
	x8t = K.quant_fp8(x.detach(), rows=False, transposed=True)[1]
	for dy in dys[::-1]:
		K.gemm_fp8(K.quant_fp8(dy, rows=False, transposed=True)[1], x8t, out=acc, epilogue=K.EPI_F32_ACC)
		bias.add_(K.colsum_(dy, torch.zeros(72, device="cuda")))
	assert torch.equal(layer.weight.main_grad, acc) and torch.equal(layer.bias.main_grad, bias)


# ------------------------------------------------------------------------------------------------ the gain's gradient
class _OneNorm(nn.Module):
	def __init__(self, d=136, n=72, tied=False):
		from elf_amd.models import NormLinear8, RMSNorm

		super().__init__()
		self.norm = NormLinear8(d, n, bias=False)
		if tied:
			self.again = RMSNorm(d)
			self.again.weight = self.norm.gamma
		self.tied = tied

	def forward(self, a):
		if self.tied:
			a = self.again(a)
		h, y = self.norm(a)
		return (h + F.pad(y, (0, 64)),)


def _norm_stage(tied, n_mb, T, g, variant="plain"):
	from elf_amd.execution import AutogradStageBlock
	from elf_amd.partitioners.utils import Signature
	from elf_amd.scheduling import OpOptions

	model = _OneNorm(tied=tied).to(torch.bfloat16)
	with torch.no_grad():
		model.norm.weight.copy_(torch.randn(72, 136, generator=torch.Generator().manual_seed(31)) * 0.05)
	ref = copy.deepcopy(model).float().cuda()
	blk = AutogradStageBlock(model, 1, [0, 1, 2], Signature(["a"], ["u"], [0], [[2]]))
	data = [(rnd(g, T, 136), rnd(g, T, 136, by=0.1).abs()) for _ in range(n_mb)]
	blk.zero_grad()
	for m, (a, dy) in enumerate(data):
		blk.input_variables[0].set(blk.input_variables[0].to_process, m, (None, a.clone()))
		blk.forward(m)
		out = blk.output_variables[0][0]
		out.get(out.to_send, m)
		out.set(out.to_process, m, (None, dy))
		if variant == "full_bwd":
			blk.backward_inputs(m, **{OpOptions.RECOMPUTE_ACTIVATIONS: True, OpOptions.RECOMPUTE_GRADIENTS: True})
			blk.recompute_forward(m, **{OpOptions.SAVE: True})
			blk.recompute_backward_inputs(m)
		else:
			blk.backward_inputs(m)
		blk.input_variables[0].get(blk.input_variables[0].to_send, m)
		blk.backward_params(m)
	return blk, ref, data


@pytest.mark.parametrize("variant", ["plain", "full_bwd"])
def test_gain_over_many_micro_batches(variant):
	"""The gain's gradient of each micro-batch is an fp32 number; their sum is that in fp32, rounded once: n half steps of fp32 and one of bf16."""
	from elf_amd import kernels as K

	n_mb, g = 96, gen(30)
	blk, _, data = _norm_stage(False, n_mb, 40, g, variant)
	norm = blk.model.norm
	_, w8t = K.quant_fp8_weight(norm.weight.detach(), rows=False, transposed=True)
	total, size, acc = torch.zeros(136, dtype=torch.float64, device="cuda"), torch.zeros(136, dtype=torch.float64, device="cuda"), torch.zeros(136, device="cuda")
	for a, dy in data:
		h, _, stats = K.rms_norm_fp8(a, norm.gamma.detach())
		one = torch.zeros(136, device="cuda")
		K.norm_bwd(K.NORM_RMS, K.gemm_fp8(K.quant_fp8(dy[:, :72].contiguous())[0], w8t), h, norm.gamma.detach(), stats, one)
		total, size = total + one.double(), size + one.double().abs()
		acc.add_(one)
	assert torch.equal(norm.gamma.main_grad, acc)
	off = n_mb * 2.0**-24 * size
	assert ((acc.double() - total).abs() <= off).all()
	blk.scale_grads(n_mb)
	assert norm.gamma.grad.dtype == torch.bfloat16
	assert ((norm.gamma.grad.double() - total / n_mb).abs() <= 2.0**-8 * (total.abs() / n_mb) + 2 * off / n_mb).all()
	blk.zero_grad()
	assert norm.gamma.grad is None and not norm.gamma.main_grad.any()


def test_gain_that_another_module_shares():
	"""A plain norm with the same parameter: both parts of its gradient count."""
	blk, ref, data = _norm_stage(True, 3, 40, gen(32))
	for a, dy in data:
		ref(a.float().requires_grad_(True))[0].backward(dy.float())
	blk.scale_grads(3)
	near(blk.model.norm.gamma.grad, ref.norm.gamma.grad / 3, 0.06, "gain")


def test_frozen_gain():
	from elf_amd.models import NormLinear8

	g = gen(33)
	layer = make(NormLinear8, 64, 48, False, E4M3, g)
	layer.gamma.requires_grad_(False)
	h, y = layer(rnd(g, 20, 64).requires_grad_(True))
	y.backward(rnd(g, 20, 48))
	moved(layer, 0)
	layer.backward(0)
	assert layer.gamma.grad is None and getattr(layer.gamma, "main_grad", None) is None


# ------------------------------------------------------------------------------------------------ one use in a forward
@pytest.mark.parametrize("which", [0, 1])
def test_only_one_of_two_uses_has_a_gradient(which):
	"""W has the input of the last use: it refuses a gradient of the first, and is right with one of the last."""
	from elf_amd import kernels as K
	from elf_amd._lib import ElfStageError
	from elf_amd.models import Linear8

	g = gen(40)
	layer = make(Linear8, 72, 48, False, E4M3, g)
	xs, dy = [rnd(g, 20, 72).requires_grad_(True) for _ in range(2)], rnd(g, 20, 48)
	ys = [layer(x) for x in xs]
	ys[which].backward(dy)
	moved(layer, 0)
	if which == 0:
		with pytest.raises(ElfStageError, match="several times"):
			layer.backward(0)
		return
	layer.backward(0)
	x8t, dy8t = (K.quant_fp8(t, rows=False, transposed=True)[1] for t in (xs[1].detach(), dy))
	assert torch.equal(layer.weight.main_grad, K.gemm_fp8(dy8t, x8t, epilogue=K.EPI_F32_STORE))


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_outside_of_a_stage(reentrant):
	"""The forward that a checkpoint runs again is no second use; neither is a call without gradients before or after the step."""
	from elf_amd.models import Linear8
	from torch.utils.checkpoint import checkpoint

	g = gen(41)
	layers = nn.Sequential(make(Linear8, 72, 48, True, E4M3, g), nn.Tanh(), make(Linear8, 48, 72, False, E5M2, g))
	x, dy = rnd(g, 20, 72), rnd(g, 20, 72)

	def step(call):
		a = x.clone().requires_grad_(True)
		with torch.no_grad():
			layers(a)
		y = call(a)
		y.backward(dy)
		for layer in (layers[0], layers[2]):
			layer.weight.main_grad = None
			moved(layer, 0)
			layer.backward(0)
		with torch.no_grad():
			layers(a)
		return y.detach(), a.grad, layers[0].weight.main_grad, layers[2].weight.main_grad

	for got, want in zip(step(lambda a: checkpoint(layers, a, use_reentrant=reentrant)), step(layers)):
		assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------ outputs written in place
@pytest.mark.parametrize("shape", [(72,), (20, 72), (2, 10, 72), (2, 3, 4, 72)])
def test_outputs_are_written_in_place(shape):
	"""``nn.ReLU(inplace=True)`` and the like behind a product give what they give on a copy."""
	from elf_amd.models import Linear8, NormLinear8

	g = gen(50)
	linear, norm = make(Linear8, 72, 48, True, E4M3, g), make(NormLinear8, 72, 48, True, E4M3, g)
	x, r, dy = rnd(g, *shape), rnd(g, *shape), rnd(g, *shape[:-1], 48)

	def step(call, change):
		a, b = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
		y = change(call(a, b))
		y.backward(dy)
		linear.clear()
		norm.clear()
		return y.detach(), a.grad

	for call in (lambda a, b: linear(a), lambda a, b: norm(a)[1], lambda a, b: norm(a, b)[1]):
		for got, want in zip(step(call, lambda y: y.mul_(2).relu_()), step(call, lambda y: y.clone().mul_(2).relu_())):
			assert got.shape == want.shape and torch.equal(got, want)


@pytest.mark.parametrize("shape", [(20, 72), (2, 10, 72)])
def test_residual_stream_written_in_place_is_refused(shape):
	"""B reads h: autograd notices that it is no longer there, whether h is the sum or the input itself."""
	from elf_amd.models import NormLinear8

	g = gen(51)
	norm = make(NormLinear8, 72, 72, False, E4M3, g)
	for inputs in ([rnd(g, *shape), rnd(g, *shape)], [rnd(g, *shape)]):
		h, y = norm(*[(t.requires_grad_(True) * 1) for t in inputs])
		h += y
		with pytest.raises(RuntimeError, match="modified by an inplace operation"):
			h.sum().backward()
		norm.clear()


def test_norm_into_given_memory():
	from elf_amd import kernels as K
	from elf_amd._lib import ElfStageError

	g = gen(52)
	x, r, gamma = rnd(g, 20, 72), rnd(g, 20, 72), 1 + rnd(g, 72, by=0.1)
	want = K.rms_norm_fp8(x, gamma, residual=r)
	for h in (torch.full_like(x, 3.0), x.clone(), r.clone()):
		into = [x.clone(), r.clone()]
		for i, t in enumerate((x, r)):
			if torch.equal(h, t):
				into[i] = h
		got = K.rms_norm_fp8(into[0], gamma, residual=into[1], h=h)
		assert got[0] is h and torch.equal(h, want[0]) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip((got[1].q, got[1].scale), (want[1].q, want[1].scale))) and torch.equal(got[2], want[2])
	with pytest.raises(ElfStageError, match="h must be dense"):
		K.rms_norm_fp8(x, gamma, residual=r, h=torch.empty(20, 80, dtype=torch.bfloat16, device="cuda")[:, :72])
	both = rnd(g, 21, 72)
	for x2, r2, h2 in ((both[:20], r, both[1:]), (x, both[1:], both[:20])):
		with pytest.raises(ElfStageError, match="shifted"):
			K.rms_norm_fp8(x2, gamma, residual=r2, h=h2)
	with pytest.raises(ElfStageError, match="x itself"):
		K.rms_norm_fp8(x, gamma, h=torch.empty_like(x))


@pytest.mark.parametrize("over", ["x", "residual"])
@pytest.mark.parametrize("T,d", [(5, 72), (7, 520), (130, 1600), (9, 4096), (67, 4104), (300, 8192)])
def test_norm_over_its_inputs(T, d, over):
	"""h in the memory of x or of the residual, at every number of chunks a thread holds."""
	from elf_amd import kernels as K

	g = gen(T + d)
	x, r, gamma = rnd(g, T, d), rnd(g, T, d), 1 + rnd(g, d, by=0.1)
	want = K.rms_norm_fp8(x, gamma, residual=r)
	got = K.rms_norm_fp8(x, gamma, residual=r, h=x if over == "x" else r)
	assert got[0] is (x if over == "x" else r) and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
	assert torch.equal(got[1].q.view(torch.uint8), want[1].q.view(torch.uint8)) and torch.equal(got[1].scale.view(torch.uint8), want[1].scale.view(torch.uint8))


# ------------------------------------------------------------------------------------------------ captured
class _Mixed(nn.Module):
	def __init__(self, d=128):
		from elf_amd.models import Linear8, NormLinear8, RMSNorm

		super().__init__()
		self.norm, self.inner, self.down, self.plain = RMSNorm(d), NormLinear8(d, 200), Linear8(200, d), nn.Linear(d, d)

	def forward(self, x):
		h, y = self.inner(self.norm(x), x)
		return h + self.plain(self.down(F.gelu(y)))


@pytest.mark.parametrize("scheduler,placement", [("afab", [0, 0]), ("afab", [0])])
def test_captured_step_of_generic_stages(scheduler, placement):
	"""Replays give what eager steps give, for the parameters of every kind of layer, with eager steps, ``zero_grad`` and other
	allocations in between."""
	from elf_amd.pipeline import Pipeline

	torch.manual_seed(60)
	stages = [_Mixed().to(torch.bfloat16) for _ in placement]
	g, mb, n_mb = gen(61), 64, 4
	draw = lambda: (rnd(g, mb * n_mb, 128), rnd(g, mb * n_mb, 128))

	def loss_fn(pred, target, reduction="sum"):
		return F.mse_loss(pred.float(), target.float(), reduction=reduction)

	x, tgt = draw()
	pipe = Pipeline(stages, x[:mb], scheduler=scheduler, partitioner=False, placement=placement)
	pipe.zero_grad()
	replay = pipe.capture_step(x, tgt, loss_fn, split_size=mb)
	for rep in range(4):
		x, tgt = draw()
		pipe.zero_grad()
		others = [torch.full((n,), 7.0, dtype=torch.bfloat16, device="cuda") for n in (128, 200, 72, 128 * 128)]  # (where given-up gradients lay)
		out, loss = replay(x, tgt)
		torch.cuda.synchronize()
		got = [t.clone() for t in out] + [p.grad.clone() for p in pipe.parameters()]
		got_main = [None if getattr(p, "main_grad", None) is None else p.main_grad.clone() for p in pipe.parameters()]
		assert all((t == 7).all() for t in others)
		pipe.zero_grad()
		want_out, want_loss = pipe(x, tgt, loss_fn, split_size=mb)
		assert float(loss) == pytest.approx(float(want_loss), rel=1e-4)
		want = [t.cuda() for t in want_out] + [p.grad for p in pipe.parameters()]
		names = [f"out {i}" for i in range(len(out))] + [n for n, _ in pipe.named_parameters()]
		for a, b, name in zip(got, want, names):
			assert torch.equal(a, b), f"replay {rep}: {name}"
		for a, p in zip(got_main, pipe.parameters()):
			assert a is None or torch.equal(a, p.main_grad), f"replay {rep}"
