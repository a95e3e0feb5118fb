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
