"""The results of K2 and K3 bit for bit: which of their products are rounded before they are added and which go into a fused multiply-add is
part of them (some outputs differ by a last bit otherwise), and no compiler option may change it.  K3's
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


def rotated(n, rope, unfused):
    """n [rows, cols] bf16, rope [rows, 256]: cosines, then sines; `unfused`: the pairs (of four in a row) that are."""
    rows, cols = n.shape
    n = n.float().view(rows, cols // 128, 16, 4, 2)
    c, s = (t.reshape(rows, 1, 16, 4, 2) for t in (rope[:, :128], rope[:, 128:]))
    re, im, c0, c1, s0, s1 = n[..., 0], n[..., 1], c[..., 0], c[..., 1], s[..., 0], s[..., 1]

    def fma(a, b, d):                                       # (a bf16 value times fp32: exact in 64 bits)
        return (a.double() * b.double() + d.double()).float()

    apart = torch.stack([re * c0 - im * s0, im * c1 + re * s1], -1)
    fused = torch.stack([fma(re, c0, -(im * s0)), fma(im, c1, re * s1)], -1)
    apart, fused = apart.to(BF), fused.to(BF)
    keep = torch.tensor([p in unfused for p in range(4)]).view(1, 1, 1, 4, 1)
    return torch.where(keep, apart, fused).view(rows, cols)


def test_rotary_embedding_bits():
    rows, heads = 32768, 2
    g = torch.Generator("cpu").manual_seed(1)
    rope = torch.randn(rows, 256, generator=g)
    wq, wk = (torch.randn(128, generator=g).to(BF) for _ in range(2))
    q, k = ((torch.randint(0, 2, (rows, heads * 128), generator=g) * 2 - 1).to(BF) for _ in range(2))
    # rows of +-1: the norm leaves them as they are, whatever its last bits
    want = [rotated(t.float() * w.float().repeat(heads), rope, (3,)) for t, w in ((q, wq), (k, wk))]
    for t, w, o in ((q, wq, want[0]), (k, wk, want[1])):    # (the case tells each pair's two ways apart)
        for p in ((), (0, 3), (1, 3), (2, 3)):
            assert (rotated(t.float() * w.float().repeat(heads), rope, p) != o).sum() > 0
    rope, wq, wk = rope.to(DEV), wq.to(DEV), wk.to(DEV)
    q1, k1, v = q.to(DEV), k.to(DEV), q.to(DEV)
    pack = ops.qk_rmsnorm_rope_pack(q1, k1, v, wq, wk, rope, rows, heads, 1, 1)
    pack = pack.view(rows, 3, heads * 128)
    ops.qk_rmsnorm_rope_(q1, k1, wq, wk, rope, rows, heads)
    for i, t in enumerate((q1, k1)):
        assert (t.cpu() != want[i]).sum() == 0 and (pack[:, i].cpu() != want[i]).sum() == 0
    # the GEMM's epilogue: every q row is the first row of +-1, every k row the second
    a = torch.zeros(rows, 64, dtype=BF)
    a[:, 0] = 1
    w = torch.zeros(2 * heads * 128, 64, dtype=BF)
    w[:, 0] = torch.cat([q[0], k[1]])
    out = ops.gemm_qknorm(a.to(DEV), w.to(DEV), None, torch.empty(rows, 2 * heads * 128, dtype=BF, device=DEV), wq, wk, rope, rows, 0,
                          heads * 128, heads)
    q1, k1 = q[:1].to(DEV).repeat(rows, 1), k[1:2].to(DEV).repeat(rows, 1)
    ops.qk_rmsnorm_rope_(q1, k1, wq, wk, rope, rows, heads)
    want = [rotated((t.float() * w.float().repeat(heads)).expand(rows, -1), rope.cpu(), (3,)) for t, w in ((q[:1], wq.cpu()), (k[1:2], wk.cpu()))]
    for i, t in enumerate((q1, k1)):
        assert (t.cpu() != want[i]).sum() == 0 and (out[:, i * heads * 128:(i + 1) * heads * 128].cpu() != want[i]).sum() == 0
