"""K3's results bit for bit: which of its products are rounded before they are added and which go into a fused multiply-add is
part of them (outputs of one row in some hundred differ by a last bit otherwise), and no compiler option may change it.  The
digests are those of the kernels built with the compiler's packed fp32 instructions, as they ran before those were turned off."""
import hashlib

import pytest
import torch

pytestmark = pytest.mark.gpu

from framepack_amd import ops  # noqa: E402

DEV = "cuda:0"
BF = torch.bfloat16


def values(rows, cols, seed):
    """bf16 values in [-4, 4) by integer arithmetic alone."""
    i = torch.arange(rows * cols, dtype=torch.int64) + seed * 1000003
    for _ in range(2):
        i = ((i ^ (i >> 15)) * 2246822519 + 3266489917) & 0xffffffff
    return ((i >> 16).float() / 8192 - 4).to(BF).view(rows, cols).to(DEV)


def digest(*tensors):
    d = hashlib.sha256()
    for t in tensors:
        d.update(t.contiguous().view(torch.uint8).cpu().numpy().tobytes())
    return d.hexdigest()[:16]


LAYERNORM = {
    256: ("79557f296cf5f936", "42a0bdb954e394e3", "bb78ef926efaa8f1"),
    1152: ("d08bb62acd013e3a", "b4ee23951cb9da25", "3dc42b47b39aacee"),
    4096: ("9af9287d4e1b6cfb", "fd2cf9d8a32d70e4", "f628d797574a3f45"),
}


@pytest.mark.parametrize("cols", list(LAYERNORM))
def test_layernorm_bits(cols):
    x, a, b = values((1 << 23) // cols, cols, 1), values(1, cols, 2)[0], values(1, cols, 3)[0]
    got = digest(ops.layernorm_modulate(x, a, b)), digest(ops.layernorm_affine(x, a, b)), digest(*ops.layernorm_modulate_fp8(x, a, b))
    assert got == LAYERNORM[cols]
