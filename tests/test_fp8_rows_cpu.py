"""``kernels.Fp8Rows`` as an object, without a GPU: copies and pickles have memory of their own."""

import copy
import io
import pickle

import pytest
import torch


def _matrix(made, dtype):
	from elf_amd import kernels as K

	torch.manual_seed(0)
	a = K.Fp8Rows.empty(37, 300, dtype, "cpu")
	a.memory.copy_(torch.randint(0, 120, a.memory.shape, dtype=torch.uint8))
	if made:
		return a
	q, s = torch.zeros(40, 448, dtype=torch.uint8), torch.zeros(3, 64, dtype=torch.uint8)
	q[:37, :384], s[:, :37] = a.q.view(torch.uint8), a.scale.view(torch.uint8)
	return K.Fp8Rows(q.view(dtype)[:37], s.view(torch.float8_e8m0fnu)[:, :37], 300)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("made", [True, False])
def test_copies_and_pickles(made, dtype):
	a = _matrix(made, dtype)

	def saved(x):
		f = io.BytesIO()
		torch.save(x, f)
		f.seek(0)
		return torch.load(f, weights_only=False)

	for way in (copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x)), saved, lambda x: copy.deepcopy({"kept": [x, x]})["kept"][1]):
		b = way(a)
		assert b.shape == a.shape and b.dtype == a.dtype and b.nbytes == a.nbytes and b.device == a.device
		assert torch.equal(b.q.view(torch.uint8)[:, :384], a.q.view(torch.uint8)[:, :384]) and torch.equal(b.scale.view(torch.uint8), a.scale.view(torch.uint8))
		# what the library would be handed is the copy's own memory
		assert b._args == (b.q.data_ptr(), a._args[1], b.scale.data_ptr(), a._args[3])
		assert (b._args[0] == a._args[0]) == (way is copy.copy)


def test_copy_of_a_layer_with_a_stash():
	from elf_amd.models import Linear8
	from elf_amd.zb_utils import Linear8DW

	layer = Linear8DW(Linear8(300, 8))
	layer._store_input8(_matrix(True, torch.float8_e4m3fn))
	layer.move_last_computed("input", 0)
	rows = copy.deepcopy(layer).ctx["input"][0].rows
	assert rows._args[0] == rows.q.data_ptr() != layer.ctx["input"][0].rows._args[0]
