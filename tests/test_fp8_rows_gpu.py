"""Matrices in 8 bits that users make themselves: every scale that the type has."""

import pytest
import torch

from tests.test_fp8_gpu import E4M3, E5M2, stands_for

pytestmark = pytest.mark.gpu


def matrix(K, dtype, byte, T=40, C=300):
	"""Values of every exponent and sign; the second block has the scale `byte`, the others 2^0 and 2^3."""
	bits = torch.arange(T * 384, device="cuda").mul_(37).remainder_(256).to(torch.uint8).view(T, 384)
	q = bits.view(dtype).float()
	bits = torch.where(torch.isfinite(q), bits, torch.zeros_like(bits))
	bits[:, C:] = 0
	s = torch.full((3, 48), 127, dtype=torch.uint8, device="cuda")
	s[2], s[1, :T] = 130, byte
	return K.Fp8Rows(bits.view(dtype), s.view(torch.float8_e8m0fnu)[:, :T], C)


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("byte", [0, 1, 100, 200, 234, 255])
def test_scales_of_every_size(byte, dtype):
	from elf_amd import kernels as K

	a = matrix(K, dtype, byte)
	want = stands_for(a)
	if byte == 255:
		want[:, 128:256] = float("nan")
	bf16 = want.float().to(torch.bfloat16)  # (2^-143 and up are fp32 numbers)
	back = K.dequant_fp8(a)
	assert torch.equal(torch.isnan(back), torch.isnan(bf16)) and torch.equal(back.nan_to_num(nan=0.0), bf16.nan_to_num(nan=0.0))
	t = K.transpose_fp8(a)
	got = stands_for(t).T
	assert torch.equal(torch.isnan(got), torch.isnan(want))
	got, want = got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0)
	# the new block's scale is 2^e for a largest value of at most 2^(e + 9) (e5m2: 2^(e + 16)) and 2^-126 at least; a value is off by half a step of its own or of the smallest normal number's
	bits, low, top = (3, -6, 9) if dtype == E4M3 else (2, -14, 16)
	exp = torch.frexp(want.abs().amax(0, keepdim=True))[1]
	step = torch.exp2((exp - top + 1).clamp_min(-126).double() + low - bits)
	assert ((got - want).abs() <= torch.maximum(want.abs() * 2.0 ** -(bits + 1), step / 2)).all()


def test_product_with_a_scale_that_is_no_number():
	from elf_amd import kernels as K

	a = matrix(K, E4M3, 127)
	s = a.scale.view(torch.uint8).clone()
	scales = torch.full((3, 48), 127, dtype=torch.uint8, device="cuda")
	scales[:, :40] = s
	scales[1, 7] = 255
	a = K.Fp8Rows(a.q, scales.view(torch.float8_e8m0fnu)[:, :40], 300)
	b = K.quant_fp8(torch.ones(50, 300, dtype=torch.bfloat16, device="cuda"))[0]
	got, back = K.gemm_fp8(a, b), K.dequant_fp8(a)
	assert torch.isnan(got[7]).all() and torch.isnan(got).sum() == 50
	assert torch.isnan(back[7, 128:256]).all() and torch.isnan(back).sum() == 128
