"""The split-backward operator plug-in of the reference (elf/zb_utils.py) on the HIP GEMM.

``LinearDX`` / ``LayerDW`` / ``LinearDW`` / ``MappingDW`` / ``replace_layer_with_layer_dw`` keep the
reference's names, queues and call order (elf/zb_utils.py:9-40, 43-194, 198-256, 487-513):

* forward   ``LinearDX.forward``  : Y = X W^T (+ b) and the input is stashed  -> ``elf_gemm_bf16`` (A, B k-contiguous)
* B         ``LinearDX.backward`` : the incoming gradient is stashed (summed when the module is used
                                    several times) and dX = dY W is returned    -> ``elf_gemm_bf16`` (B reduction-major)
* W         ``LinearDW.backward`` : dW += dY^T X, db += sum_t dY                -> ``elf_gemm_bf16`` (both reduction-major,
                                    fp32 ``C +=``) and ``elf_colsum_bf16``

Differences from the reference, both on purpose: gradients accumulate in fp32 buffers
(``weight.main_grad`` / ``bias.main_grad``; ``weight.grad`` is only written by a block's ``scale_grads``)
instead of in the parameter dtype, and there is no other execution path: a ``LinearDW`` must be bf16 on
the GPU with ``in_features`` and ``out_features`` multiples of 64, and the tokens of a call a
multiple of 64 (the GEMM's tile constraints) - anything else raises.

``Linear8`` and ``NormLinear8`` layers (elf_amd.models) are replaced by ``Linear8DW`` and ``NormLinear8DW``, the same split in 8 bits,
which the reference does not have.
"""

import torch
import torch.nn as nn

from . import _lib, kernels
from .models import Linear8, NormLinear8

__all__ = ["LinearDX", "LayerDW", "LinearDW", "Linear8DX", "Linear8DW", "NormLinear8DX", "NormLinear8DW", "MappingDW", "replace_layer_with_layer_dw", "replace_linear_with_linear_dw"]


def _as_rows(t):
	"""[..., C] -> contiguous [rows, C] (a copy only if the layout forces one)."""
	if t.dim() == 2 and t.is_contiguous():
		return t
	t2 = t.reshape(-1, t.shape[-1])
	return t2 if t2.is_contiguous() else t2.contiguous()


class LinearDX(torch.autograd.Function):
	"""y = linear(x) whose backward only computes the input gradient (elf/zb_utils.py:9-40)."""

	@staticmethod
	def forward(ctx, input, weight, bias, linear):
		ctx.linear = linear
		linear._store_input(input)
		ctx.save_for_backward(input.detach())  # marks the input as needed by the backward, so that torch.utils.checkpoint recomputes it
		x = _as_rows(input)
		if bias is not None:
			# one dense row of N values as it lies (the views take 3 us); expand refuses any other size but 1
			row = bias if bias.numel() == weight.shape[0] and bias.is_contiguous() else bias.reshape(1, -1).expand(1, weight.shape[0]).contiguous()
			y = kernels.gemm(x, weight, epilogue=kernels.EPI_BF16_RESID, residual=row, residual_ld=0)
		else:
			y = kernels.gemm(x, weight)
		return y if input.dim() == 2 else y.view(*input.shape[:-1], weight.shape[0])

	@staticmethod
	def backward(ctx, grad_output):
		linear = ctx.linear
		linear._accumulate_grad_output(grad_output)
		go = _as_rows(grad_output)
		grad_input = kernels.gemm(go, linear.weight.detach(), b_t=True)  # dY [T, out] x W [out, in] with W read as it lies
		return (grad_input if grad_output.dim() == 2 else grad_input.view(*grad_output.shape[:-1], linear.weight.shape[1])), None, None, None


class LayerDW:
	"""Mixin for modules whose backward is split: an autograd function that only produces the input
	gradient and stashes what the parameter gradient needs, and ``backward(mb_id)`` that consumes the
	stash (elf/zb_utils.py:43-194).  ``ctx["input"]`` / ``ctx["grad_output"]`` are per-micro-batch lists."""

	_dx_function_registry = {}

	def __init__(self, *args, **kwargs):
		with torch.device("meta"):  # the tensors are replaced by the wrapped layer's right away
			super().__init__(*args, **kwargs)
		self.ctx = {"input": [], "grad_output": []}
		self.last_input = None
		self.last_grad_output = None

	@classmethod
	def register_dx_function(cls, dx_class):
		cls._dx_function_registry[cls] = dx_class
		return dx_class

	def backward(self, mb_id):
		raise NotImplementedError("Subclasses must implement backward()")

	def clear(self):
		self.ctx["input"].clear()
		self.ctx["grad_output"].clear()
		self.last_input = None
		self.last_grad_output = None

	def is_empty(self, queue):
		return all(x is None for x in self.ctx[queue])

	def _state(self):
		return f"({sum(x is not None for x in self.ctx['input'])},{sum(x is not None for x in self.ctx['grad_output'])})"

	# (last_input and last_grad_output are plain attributes: nn.Module.__setattr__ first looks for a parameter, a module and a
	# buffer of that name, 3 us each time)
	def _store_input(self, input):
		last = input.detach()
		# an input without a grad_fn is the stage's own input: checkpointing will not recompute it, so the
		# remat logic must not drop it
		last.is_model_input = input.grad_fn is None
		self.__dict__["last_input"] = last

	def _accumulate_grad_output(self, grad_output):
		last = getattr(self, "last_grad_output", None)
		self.__dict__["last_grad_output"] = grad_output if last is None else last + grad_output

	def set(self, queue, idx, value):
		values = self.ctx[queue]
		if len(values) <= idx:
			values.extend([None] * (idx - len(values) + 1))
		if values[idx] is not None:
			raise ValueError(f"{queue} at index {idx} already set")
		values[idx] = value

	def delete(self, queue, idx):
		values = self.ctx[queue]
		if idx >= len(values) or values[idx] is None:
			raise ValueError(f"{queue} at index {idx} not set")
		values[idx] = None

	def move_last_computed(self, queue, idx):
		last_value = getattr(self, f"last_{queue}", None)
		if last_value is None:
			return  # a sub-module the forward did not use
		self.set(queue, idx, last_value)
		self.__dict__[f"last_{queue}"] = None

	def offload_last(self, idx, to="cpu"):
		with torch.no_grad():
			self.ctx["grad_output"][idx] = self.ctx["grad_output"][idx].to(to, non_blocking=True)
			self.ctx["input"][idx] = self.ctx["input"][idx].to(to, non_blocking=True)


class LinearDW(LayerDW, nn.Linear):
	"""``nn.Linear`` with the split backward (elf/zb_utils.py:198-256), sharing the wrapped layer's
	parameters.  Call order: LinearDW.forward -> LinearDX.forward -> LinearDX.backward -> LinearDW.backward."""

	def __init__(self, linear, *args, **kwargs):
		if linear.in_features % 64 or linear.out_features % 64:
			raise _lib.ElfStageError(f"LinearDW: in_features and out_features must be multiples of 64 for the HIP GEMM, got {linear.in_features} -> {linear.out_features}")
		super().__init__(linear.in_features, linear.out_features, linear.bias is not None, *args, **kwargs)
		self.weight = linear.weight
		if linear.bias is not None:
			self.bias = linear.bias

	def _check(self, x):
		if x.dtype != torch.bfloat16 or not x.is_cuda or self.weight.dtype != torch.bfloat16 or not self.weight.is_cuda:
			raise _lib.ElfStageError(f"LinearDW: bf16 tensors on the GPU only (input {x.dtype} on {x.device}, weight {self.weight.dtype} on {self.weight.device})")
		if (x.numel() // x.shape[-1]) % 64:
			raise _lib.ElfStageError(f"LinearDW: the number of tokens of a call must be a multiple of 64, got input {tuple(x.shape)}")

	def forward(self, x, *args, **kwargs):
		self._check(x)
		return LinearDX.apply(x, self.weight, self.bias, self, *args, **kwargs)

	def _main_grad(self, param):
		g = getattr(param, "main_grad", None)
		if g is None:
			g = torch.zeros(param.shape, dtype=torch.float32, device=param.device)
			param.main_grad = g
		return g

	def backward(self, mb_id):
		"""W: main_grad += dY^T X (fp32), bias main_grad += sum over tokens of dY; drops the stash."""
		grad_output = self.ctx["grad_output"][mb_id]
		inputs = self.ctx["input"][mb_id]
		go, inp = _as_rows(grad_output), _as_rows(inputs)
		kernels.gemm(go, inp, a_t=True, b_t=True, out=self._main_grad(self.weight), epilogue=kernels.EPI_F32_ACC)
		if self.bias is not None:
			kernels.colsum_(go, self._main_grad(self.bias))
		self.ctx["grad_output"][mb_id] = None
		self.ctx["input"][mb_id] = None

	_own_backward = backward  # what backward_together stands for: a method put in its place, on the class too, is asked layer by layer

	@staticmethod
	def backward_together(layers, mb_id):
		"""W of several layers: what ``backward`` does for each, the layers over the same number of tokens in one call of the library
		(weight gradients and bias sums then share launches).  What such a call does not take goes through ``backward``, and so do layers whose
		stash has to be copied to dense rows: one copy is alive at a time."""
		by_tokens = {}
		for m in layers:
			grad_output, inputs, acc = m.ctx["grad_output"][mb_id], m.ctx["input"][mb_id], m._main_grad(m.weight)
			bias = m._main_grad(m.bias) if m.bias is not None else None
			if not all(g is None or (g.dtype == torch.float32 and g.is_contiguous()) for g in (acc, bias)) or not all(t.dtype == torch.bfloat16 and t.is_contiguous() for t in (grad_output, inputs)):
				m.backward(mb_id)
				continue
			go, inp = _as_rows(grad_output), _as_rows(inputs)
			by_tokens.setdefault(go.shape[0], []).append((m, (go, inp, acc, bias)))
		for group in by_tokens.values():
			kernels.linear_w_pass([layer for _, layer in group])
			for m, _ in group:
				m.ctx["grad_output"][mb_id] = None
				m.ctx["input"][mb_id] = None


LinearDW.register_dx_function(LinearDX)

# ------------------------------------------------------------------------------------------------ 8 bits
class _Use:
	"""One forward call of a layer in 8 bits.  ``lost``: the layer was called again before its input was moved, so W would multiply this call's
	output gradient with the other's input.  A checkpoint that runs the forward again, within a backward pass (``task``), loses nothing: it
	stores the input that was there."""

	__slots__ = ("task", "lost")

	def __init__(self):
		self.task, self.lost = torch._C._current_graph_task_id(), False


class _Kept8:
	"""What a layer in 8 bits keeps of a micro-batch: its input or its output gradient along the tokens (``kernels.Fp8Rows`` of the
	transpose: half of the bf16 bytes, with the tokens filled up to 128), and of an output gradient its sum over the tokens where there is a
	bias and the gradient of the gain where there is a norm, both in fp32.  ``use``: the forward call it belongs to; ``more``: what came
	before it of the same call (a stage goes back from its outputs one after the other)."""

	__slots__ = ("rows", "bias", "gain", "use", "more")

	def __init__(self, rows, bias=None, use=None, gain=None, more=None):
		self.rows, self.bias, self.gain, self.use, self.more = rows, bias, gain, use, more

	def to(self, device, non_blocking=False):
		def there(part):
			return None if part is None else part.to(device, non_blocking=non_blocking)

		return _Kept8(there(self.rows), there(self.bias), self.use, there(self.gain), there(self.more))


def _forward8(x8, linear, lead):
	"""[*lead, out_features] of rows in 8 bits, in memory of its own: a view would keep users from writing into it in place."""
	w8, _ = kernels.quant_fp8_weight(linear.weight.detach())
	y = rows = None
	if len(lead) != 1:
		y = torch.empty((*lead, linear.weight.shape[0]), dtype=torch.bfloat16, device=linear.weight.device)
		rows = y.view(-1, y.shape[-1])
	if linear.bias is None:
		rows = kernels.gemm_fp8(x8, w8, out=rows)
	else:
		rows = kernels.gemm_fp8(x8, w8, out=rows, epilogue=kernels.EPI_BF16_RESID, residual=linear.bias.detach(), residual_ld=0)
	return rows if y is None else y


def _backward8(go, linear, use):
	"""The input gradient of the forward call ``use``; the output gradient is kept for W."""
	dy8, dy8t = kernels.quant_fp8(go, dtype=linear.grad_dtype, transposed=True)
	bias = None
	if linear.bias is not None:
		bias = kernels.colsum_(go, torch.zeros(go.shape[1], dtype=torch.float32, device=go.device))
	linear._store_grad_output(_Kept8(dy8t, bias, use))
	_, w8t = kernels.quant_fp8_weight(linear.weight.detach(), rows=False, transposed=True)
	return kernels.gemm_fp8(dy8, w8t)


class Linear8DX(torch.autograd.Function):
	"""``LinearDX`` in 8 bits.  One read of the input makes both the product's operand and what W keeps of it; B makes the
	same two of the output gradient.  The weight goes into 8 bits in F and in B (it is read for the product anyway, and nothing
	has to know when an optimizer has changed it)."""

	@staticmethod
	def forward(ctx, input, weight, bias, linear):
		x8, x8t = kernels.quant_fp8(_as_rows(input.detach()), transposed=True)
		ctx.linear, ctx.in_shape, ctx.use = linear, input.shape, linear._store_input8(x8t)
		ctx.save_for_backward(x8t.memory)  # read again in B, so that torch.utils.checkpoint runs the forward again
		return _forward8(x8, linear, input.shape[:-1])

	@staticmethod
	def backward(ctx, grad_output):
		ctx.saved_tensors  # noqa: B018
		return _backward8(_as_rows(grad_output), ctx.linear, ctx.use).view(ctx.in_shape), None, None, None


class Linear8DW(LayerDW, Linear8):
	"""``Linear8`` with the split backward, sharing the wrapped layer's parameters: queues and call order of ``LinearDW``, any number of
	tokens and features (out_features a multiple of 8 with a bias), one use in a forward."""

	def __init__(self, linear, *args):
		super().__init__(linear.in_features, linear.out_features, linear.bias is not None, None, None, linear.grad_dtype, *args)
		if linear.bias is not None and linear.out_features % 8:
			raise _lib.ElfStageError(f"{type(self).__name__}: out_features must be a multiple of 8 where there is a bias, got {linear.out_features}")
		self.weight = linear.weight
		if linear.bias is not None:
			self.bias = linear.bias

	def _check(self, x):
		if x.dtype != torch.bfloat16 or not x.is_cuda or self.weight.dtype != torch.bfloat16 or not self.weight.is_cuda:
			raise _lib.ElfStageError(f"{type(self).__name__}: bf16 tensors on the GPU only (input {x.dtype} on {x.device}, weight {self.weight.dtype} on {self.weight.device})")

	def _store_input8(self, rows):
		last, use = self.last_input, _Use()
		if last is not None and last.use.task == use.task:
			last.use.lost = True
		self.__dict__["last_input"] = _Kept8(rows, use=use)
		return use

	def _store_grad_output(self, kept):
		last = getattr(self, "last_grad_output", None)
		if last is not None and last.use is not kept.use:
			raise _lib.ElfStageError(f"{type(self).__name__}: the layer was used several times in one forward (sums of output gradients in 8 bits would need bf16 again)")
		kept.more = last
		self.__dict__["last_grad_output"] = kept

	_main_grad = LinearDW._main_grad

	def forward(self, x):
		self._check(x)
		return Linear8DX.apply(x, self.weight, self.bias, self)

	def backward(self, mb_id):
		"""W: main_grad += dY^T X (fp32) from the two 8-bit matrices, the bias's and the gain's += what B left; drops the stash."""
		kept, x = self.ctx["grad_output"][mb_id], self.ctx["input"][mb_id]
		if kept.use.lost:
			raise _lib.ElfStageError(f"{type(self).__name__}: the layer was used several times in one forward, or again before its input was moved: what is kept is not the input of the use that has a gradient")
		while kept is not None:
			kernels.gemm_fp8(kept.rows, x.rows, out=self._main_grad(self.weight), epilogue=kernels.EPI_F32_ACC)
			if self.bias is not None:
				self._main_grad(self.bias).add_(kept.bias)
			if kept.gain is not None:
				self._main_grad(self.gamma).add_(kept.gain)
			kept = kept.more
		self.ctx["grad_output"][mb_id] = None
		self.ctx["input"][mb_id] = None


class NormLinear8DX(torch.autograd.Function):
	"""(h, y) of ``NormLinear8`` (y alone without a residual).  B reads h again: where h was written in place, autograd refuses.  It hands the
	norm's backward the product's result, in bf16 as every layer's input gradient, and h's own gradient.  The gain's gradient of a
	micro-batch goes through autograd, rounded, and is kept in fp32 for W."""

	@staticmethod
	def forward(ctx, x, residual, gamma, weight, bias, linear):
		rows, added, h = _as_rows(x.detach()), None, None
		if residual is not None:
			added, h = _as_rows(residual.detach()), torch.empty(x.shape, dtype=x.dtype, device=x.device)
		h_rows, n8, stats = kernels.rms_norm_fp8(rows, gamma.detach(), residual=added, eps=linear.eps, h=None if h is None else h.view(rows.shape))
		ctx.linear, ctx.in_shape, ctx.use, ctx.added = linear, x.shape, linear._store_input8(kernels.transpose_fp8(n8)), residual is not None
		ctx.set_materialize_grads(False)
		y = _forward8(n8, linear, x.shape[:-1])
		ctx.save_for_backward(h_rows if h is None else h, stats, gamma)
		return (h, y) if ctx.added else y

	@staticmethod
	def backward(ctx, *grads):
		dh, dy = grads if ctx.added else (None, grads[0])
		h, stats, gamma = ctx.saved_tensors
		dx, dgamma = dh, None
		if dy is not None:
			acc = torch.zeros(gamma.shape, dtype=torch.float32, device=gamma.device)
			dn = _backward8(_as_rows(dy), ctx.linear, ctx.use)
			dx = kernels.norm_bwd(kernels.NORM_RMS, dn, _as_rows(h), gamma.detach(), stats, acc, dres=None if dh is None else _as_rows(dh)).view(ctx.in_shape)
			if ctx.needs_input_grad[2]:
				dgamma = acc.to(gamma.dtype)
				if ctx.linear.gain_in_main:
					ctx.linear.last_grad_output.gain = acc
		return dx, dx if ctx.added else None, dgamma, None, None, None


class NormLinear8DW(Linear8DW, NormLinear8):
	"""``NormLinear8`` with the split backward.  in_features: a multiple of 8, at most 8192.  The gain's gradient is summed over micro-batches in W, in
	fp32 ``gamma.main_grad`` like the weight's and the bias's.  ``gamma.grad`` has it too, as autograd sums it in B: rounded to the parameter's
	type after every micro-batch, until a block's ``scale_grads`` writes it from ``main_grad``."""

	gain_in_main = True  # (a block says no where a module of another kind has the same parameter: only autograd's sum has that one's part)

	def __init__(self, linear):
		super().__init__(linear, linear.eps)
		if linear.in_features % 8 or linear.in_features > 8192:
			raise _lib.ElfStageError(f"NormLinear8DW: in_features must be a multiple of 8 and at most 8192, got {linear.in_features}")
		self.gamma = linear.gamma

	def forward(self, x, residual=None):
		self._check(x)
		if residual is None:
			return x, NormLinear8DX.apply(x, None, self.gamma, self.weight, self.bias, self)
		self._check(residual)
		if residual.shape != x.shape:
			raise _lib.ElfStageError(f"NormLinear8DW: x {tuple(x.shape)} and the residual {tuple(residual.shape)} differ in shape")
		return NormLinear8DX.apply(x, residual, self.gamma, self.weight, self.bias, self)


Linear8DW.register_dx_function(Linear8DX)
NormLinear8DW.register_dx_function(NormLinear8DX)

# module class -> its split-backward replacement (the reference also maps nn.Conv1d; convolutions are not
# part of the transformer-stage path this build covers)
MappingDW = {nn.Linear: LinearDW, Linear8: Linear8DW, NormLinear8: NormLinear8DW}


def replace_layer_with_layer_dw(model, only=None):
	"""Replace, in place, every module whose class is in ``MappingDW`` by its split-backward
	equivalent (elf/zb_utils.py:490-513)."""
	for name, module in list(model.named_modules()):
		if type(module) in MappingDW and not isinstance(module, LayerDW) and (only is None or type(module) in only):
			parent = model if "." not in name else model.get_submodule(name[: name.rfind(".")])
			setattr(parent, name.split(".")[-1], MappingDW[type(module)](module))


def replace_linear_with_linear_dw(model, device=None):
	"""Older name of ``replace_layer_with_layer_dw(model, only=[nn.Linear])`` (elf/zb_utils.py:449-485)."""
	replace_layer_with_layer_dw(model, only=[nn.Linear])
