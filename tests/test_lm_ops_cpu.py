"""What the entry points of K12 and K13 refuse, on the CPU: the tensor-level checks (the device check aside, everything
that is refused is refused before the library is called) and the C ABI's (a refused call launches nothing)."""
import pytest
import torch

from framepack_amd import lib as fplib
from framepack_amd import ops

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def no_device_check(monkeypatch):
    monkeypatch.setattr(ops, "_dev", lambda *ts: None)

    class Lib:
        def __getattr__(self, name):
            raise AssertionError("the library was called")

    monkeypatch.setattr(fplib, "load", lambda: Lib())


def mats(*shapes, dtype=BF):
    return [torch.zeros(*s, dtype=dtype) for s in shapes]


def test_cpu_tensors_are_refused():
    x, w, m = torch.zeros(4, 64, dtype=BF), torch.ones(64, dtype=BF), torch.zeros(16, 64, dtype=BF)
    for call in (lambda: ops.rmsnorm_residual(x, w), lambda: ops.rmsnorm_residual_fp8(x, w), lambda: ops.gated_ff(x, m, m),
                 lambda: ops.rmsnorm_residual_backward(x, x, w), lambda: ops.gated_ff_backward(m, x, m, m, m, m)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_norm_refusals(no_device_check):
    x, r, w = torch.zeros(4, 64, dtype=BF), torch.zeros(4, 64, dtype=BF), torch.ones(64, dtype=BF)
    big = torch.zeros(4, 200, dtype=BF)
    cases = [
        (lambda: ops.rmsnorm_residual(x.float(), w), "expected torch.bfloat16 or"),
        (lambda: ops.rmsnorm_residual(x, w.half()), "weight"),
        (lambda: ops.rmsnorm_residual(x, w[:32]), "weight"),
        (lambda: ops.rmsnorm_residual(x, w, r[:3]), "resid"),
        (lambda: ops.rmsnorm_residual(x, w, r.half()), "resid"),
        (lambda: ops.rmsnorm_residual(x[0], w), "rows, cols"),
        (lambda: ops.rmsnorm_residual(x.t(), w), "unit inner stride"),
        (lambda: ops.rmsnorm_residual(torch.zeros(4, 128, dtype=BF)[:, ::2], w), "unit inner stride"),
        (lambda: ops.rmsnorm_residual(torch.zeros(4, 0, dtype=BF), w[:0]), "column"),
        (lambda: ops.rmsnorm_residual(x, w, eps=-1.0), "eps"),
        (lambda: ops.rmsnorm_residual(x[:1].expand(2 ** 32 + 4, 64), w), "more than"),
        (lambda: ops.rmsnorm_residual(x, w, eps=float("nan")), "eps"),
        (lambda: ops.rmsnorm_residual(x, w, resid_out=r), "without resid"),
        (lambda: ops.rmsnorm_residual(x, w, r, out=torch.zeros(4, 32, dtype=BF)), "out"),
        (lambda: ops.rmsnorm_residual(x, w, r, out=x[:1].expand(4, 64)), "overlap"),
        (lambda: ops.rmsnorm_residual(x, w, r, out=x, resid_out=x), "share memory"),
        (lambda: ops.rmsnorm_residual(big[:, :64], w, r, out=big[:, 8:72]), "shares memory"),
        (lambda: ops.rmsnorm_residual(big[:3, :64], w, out=big[1:, :64]), "shares memory"),
        (lambda: ops.rmsnorm_residual(x, w, out=w[None].expand(4, 64)), "overlap"),
        (lambda: ops.rmsnorm_residual(x[:1], w, out=w[None]), "shares memory"),
        (lambda: ops.rmsnorm_residual_fp8(x.half(), w.half()), "x"),
        (lambda: ops.rmsnorm_residual_fp8(x, w, out=r), "out"),
        (lambda: ops.rmsnorm_residual_fp8(x, w, out_scale=torch.zeros(3)), "out_scale"),
        (lambda: ops.rmsnorm_residual_fp8(x, w, out_scale=torch.zeros(8)[::2]), "out_scale"),
        (lambda: ops.rmsnorm_residual_fp8(x, w, out=x.view(ops.FP8)[:, :64]), "shares memory"),
        (lambda: ops.rmsnorm_residual_backward(x, r[:3], w), "dy"),
        (lambda: ops.rmsnorm_residual_backward(x, r, w, dh=r[:, :32]), "dh"),
        (lambda: ops.rmsnorm_residual_backward(x, r, w, dx=x), "shares memory"),
        (lambda: ops.rmsnorm_residual_backward(x, r, w, dx=r), "shares memory"),
        (lambda: ops.rmsnorm_residual_backward(x.half(), r, w), "dy"),
    ]
    for call, text in cases:
        with pytest.raises(ValueError, match=text):
            call()


def test_gated_ff_refusals(no_device_check):
    x, wg, wu, b = torch.zeros(4, 64, dtype=BF), torch.zeros(16, 64, dtype=BF), torch.zeros(16, 64, dtype=BF), torch.zeros(16, dtype=BF)
    g, u, dh = mats((4, 16), (4, 16), (4, 16))
    x8, w8, s4, s16 = torch.zeros(4, 128, dtype=ops.FP8), torch.zeros(16, 128, dtype=ops.FP8), torch.ones(4), torch.ones(16)
    cases = [
        (lambda: ops.gated_ff(x.float(), wg.float(), wu.float()), "x"),
        (lambda: ops.gated_ff(x, wg.half(), wu), "w_gate"),
        (lambda: ops.gated_ff(x, wg, wu[:8]), "w_up"),
        (lambda: ops.gated_ff(x, wg[:, :32], wu), "w_gate"),
        (lambda: ops.gated_ff(x, wg[:0], wu[:0]), "row"),
        (lambda: ops.gated_ff(x, wg.t().contiguous().t(), wu), "unit inner stride"),
        (lambda: ops.gated_ff(x, wg, wu, b, None), "both or neither"),
        (lambda: ops.gated_ff(x, wg, wu, b, b[:8]), "b_up"),
        (lambda: ops.gated_ff(x, wg, wu, b.float(), b.float()), "b_gate"),
        (lambda: ops.gated_ff(x, wg, wu, act=2), "act"),
        (lambda: ops.gated_ff(x, wg, wu, out=g[:, :8]), "out"),
        (lambda: ops.gated_ff(x, wg, wu, out=g[:1].expand(4, 16)), "overlap"),
        (lambda: ops.gated_ff(x, wg, wu, out=x[:, :16]), "shares memory"),
        (lambda: ops.gated_ff_fp8(x, s4, wg, s16, wu, s16), "x"),
        (lambda: ops.gated_ff_fp8(x8, s4[:3], w8, s16, w8, s16), "x_scale"),
        (lambda: ops.gated_ff_fp8(x8, s4, w8, s16.half(), w8, s16), "wg_scale"),
        (lambda: ops.gated_ff_fp8(x8, s4, w8, s16, w8, s16, out=g.half()), "out"),
        (lambda: ops.gated_ff_backward(dh[:3], x, wg, wu, g, u), "dh"),
        (lambda: ops.gated_ff_backward(dh, x, wg, wu, g, u[:, :8]), "up"),
        (lambda: ops.gated_ff_backward(dh, x, wg, wu, g.half(), u), "gate"),
        (lambda: ops.gated_ff_backward(dh, x, wg, wu, g, u, act=None), "act"),
    ]
    for call, text in cases:
        with pytest.raises(ValueError, match=text):
            call()


def test_disjoint_columns_and_rows_of_one_buffer_do_not_share():
    big = torch.zeros(10, 96, dtype=BF)
    a, b = big[:, :32], big[:, 32:64]
    assert not ops._share(a, b) and not ops._share(b, a) and not ops._share(big[:5], big[5:])
    assert ops._share(big[:, :33], b) and ops._share(b, big[:, :33]) and ops._share(big[:6], big[5:]) and ops._share(a, a)
    assert ops._share(big[1:, 80:], big.view(-1)[90:90 + 96].view(1, 96)) is True
    assert not ops._share(big[:1, :8], big[:, 8:]) and not ops._share(big[:, 8:], big[9:, :8])
    assert not ops._share(big[:0], big) and ops._share(big[:1].expand(4, 96), big)


def test_the_library_refuses_without_launching():
    L = fplib.load()
    p, n, m = 1 << 20, 4, 64                                # addresses that nothing may touch

    def refused(name, *a):
        assert getattr(L, name)(*a) == 1, (name, a)

    ok = [p, m, p, m, p, p, m, p, m, n, m, 1e-6, None]
    for name in ("fp_rmsnorm_residual_bf16", "fp_rmsnorm_residual_f16"):
        for i, v in ((0, None), (4, None), (5, None), (1, -1), (3, -1), (6, m - 1), (8, m - 1), (9, -1), (10, 0), (11, -1.0),
                     (7, None), (2, None)):
            refused(name, *[v if j == i else t for j, t in enumerate(ok)])
        refused(name, *[p + 1 if j == 0 else t for j, t in enumerate(ok)])          # not even the type's alignment
        assert getattr(L, name)(*[0 if j == 9 else t for j, t in enumerate(ok)]) == 0          # no rows: nothing to do
    ok = [p, m, p, m, p, p, m, p, p, m, n, m, 1e-6, None]
    for i, v in ((0, None), (7, None), (7, p + 2), (5, None), (6, m - 1), (10, -1), (12, -1.0)):
        refused("fp_rmsnorm_residual_fp8", *[v if j == i else t for j, t in enumerate(ok)])
    ok = [p, m, p, m, p, m, p, p, m, p, n, m, 1e-6, p, 1 << 30, None]
    for i, v in ((0, None), (2, None), (6, None), (7, None), (9, None), (8, m - 1), (10, 0), (11, 0), (13, None), (13, p + 4), (14, 16)):
        refused("fp_rmsnorm_residual_backward_bf16", *[v if j == i else t for j, t in enumerate(ok)])
    assert L.fp_rmsnorm_residual_backward_workspace_bytes(0, 8) == 0 and L.fp_gated_ff_backward_workspace_bytes(p, 8, p, 8, p, 8, 4, 0, 8) == 0
    F, K = 16, 128
    ok = [p, K, p, K, p, K, p, p, p, F, p, p, F, n, F, K, 0, None, 0, None]
    for i, v in ((0, None), (2, None), (4, None), (8, None), (6, None), (7, None), (10, None), (9, F - 1), (12, F - 1), (3, K - 1),
                 (13, -1), (14, 0), (15, 0), (16, 2)):
        refused("fp_gated_ff_bf16", *[v if j == i else t for j, t in enumerate(ok)])
    size = L.fp_gated_ff_workspace_bytes
    assert size(p, K, p, K, p, K, 49, F, K) == 0 and size(p + 2, K, p, K, p, K, 48, F, K) == 0
    assert size(p + 2, K, p, K, p, K, 49, F, K) == 49 * K * 2 and size(p, K, p, K + 4, p, K, 49, F, K) == F * K * 2
    assert size(p, K, p, K, p, K, 49, F, K - 1) == (49 + 2 * F) * K * 2
    ok[13], ok[15] = 49, K - 1                              # a width that has to be copied: not without the space
    refused("fp_gated_ff_bf16", *ok)
    refused("fp_gated_ff_f16", *[p + 8 if j == 17 else 1 << 30 if j == 18 else t for j, t in enumerate(ok)])
    refused("fp_gated_ff_f16", *[p if j == 17 else (49 + 2 * F) * K * 2 - 1 if j == 18 else t for j, t in enumerate(ok)])
    ok = [p, K, p, p, K, p, p, K, p, p, p, p, F, n, F, K, 0, None, 0, None]
    for i, v in ((0, None), (2, None), (5, None), (8, None), (1, K + 8), (4, K + 8), (7, K + 8), (0, p + 8), (3, p + 8), (6, p + 8),
                 (11, p + 8), (12, F + 4), (14, 12), (15, 64), (5, p + 4), (9, p + 2), (9, None), (16, -1)):
        refused("fp_gated_ff_fp8", *[v if j == i else t for j, t in enumerate(ok)])
    assert L.fp_gated_ff_fp8_workspace_bytes(4, 16, 128) == 0 and L.fp_gated_ff_fp8_workspace_bytes(4, 14336, 4096) == 0
    need = L.fp_gated_ff_fp8_workspace_bytes(4, 16, 8192)                          # few columns, a long K: parts of it
    assert need > 0 and need % (4 * 2 * 16 * 4) == 0
    ok[1] = ok[4] = ok[7] = ok[15] = 8192
    for i, v in ((17, None), (17, p + 8), (18, need - 1)):
        refused("fp_gated_ff_fp8", *[v if j == i else p if j == 17 else need if j == 18 else t for j, t in enumerate(ok)])
    ok = [p, F, p, K, p, K, p, K, p, F, p, F, p, p, p, n, F, K, 0, p, 1 << 30, None]
    for i, v in ((0, None), (2, None), (4, None), (8, None), (12, None), (13, None), (5, K - 1), (7, K - 1), (12, p + 8), (13, p + 2),
                 (14, p + 1), (15, 0), (16, 0), (17, 0), (15, 1 << 20), (18, 3), (19, None), (19, p + 8), (20, 16)):
        refused("fp_gated_ff_backward_f16", *[v if j == i else t for j, t in enumerate(ok)])


def test_the_library_refuses_sizes_whose_launches_would_not_fit():
    L = fplib.load()
    p, big = 1 << 20, 1 << 28
    ok = [p, big, None, 0, p, p, big, None, 0, 1, big + 1, 1e-6, None]
    ok[1] = ok[6] = big + 8
    assert L.fp_rmsnorm_residual_bf16(*ok) == 1 and L.fp_rmsnorm_residual_f16(*ok) == 1
    assert L.fp_rmsnorm_residual_backward_workspace_bytes(1, big + 1) == 0
    ld = big + 8
    assert L.fp_rmsnorm_residual_backward_bf16(p, ld, p, ld, None, 0, p, p, ld, p, 1, big + 1, 1e-6, p, 1 << 60, None) == 1
    F = (1 << 27) + 1
    assert L.fp_gated_ff_workspace_bytes(p, 8, p, 8, p, 8, 1, F, 8) == 0
    assert L.fp_gated_ff_bf16(p, 8, p, 8, p, 8, None, None, p, F, None, None, 0, 1, F, 8, 0, None, 0, None) == 1


def test_fragment_reads_of_the_gated_blocks_products_all_feed_an_mfma(tmp_path):
    """The 16-bit instances of the 4-wave kernel read their MFMA fragments with inline asm - K13's gradient with pairs of
    transposing reads - whose results the compiler takes for written at once.  Compile K13's products to assembly with the
    Makefile's flags and check, per kernel: no register of a read in flight is touched by a compiler instruction or written
    by another read before an MFMA has taken it, every read is taken, nothing goes to scratch memory."""
    import os
    import re
    import subprocess
    hipcc = "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("needs hipcc")
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "framepack_amd", "csrc")
    mk = open(os.path.join(csrc, "Makefile")).read()
    flags = re.search(r"^CXXFLAGS = (.*)$", mk, re.M).group(1).replace("$(ARCH)", "gfx950").replace("-fPIC", "").split()
    files = ("gated_ff_mfma", "gated_ff_grad_mfma")
    procs = [subprocess.Popen([hipcc, *flags, "-S", "--cuda-device-only", os.path.join(csrc, f + ".hip"), "-o", str(tmp_path / (f + ".s"))],
                              stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL) for f in files]
    seen = transposing = 0
    for f, pr in zip(files, procs):
        assert pr.wait() == 0, f
        text = (tmp_path / (f + ".s")).read_text()
        for m in re.finditer(r"^(_ZN7fp_gemm14gemm_w4_kernel\S*):[^\n]*\n(.*?)^\s*\.amdhsa_kernel \1", text, re.S | re.M):
            name, body = m.group(1), m.group(2)
            seen += 1
            pending, in_asm = {}, False                     # register -> the read that is on its way into it
            for line in body.splitlines():
                t = line.strip()
                if "#ASMSTART" in t or "#ASMEND" in t:
                    in_asm = "#ASMSTART" in t
                    continue
                regs = {int(r) for r in re.findall(r"\bv(\d+)\b", t)}
                for lo, hi in re.findall(r"\bv\[(\d+):(\d+)\]", t):
                    regs |= set(range(int(lo), int(hi) + 1))
                rd = re.match(r"ds_read_(b128|b64_tr_b16) v\[(\d+):(\d+)\], v(\d+)", t) if in_asm else None
                if rd:
                    assert not regs & set(pending), (name, "a fragment read is overwritten before any MFMA used it", t)
                    transposing += rd.group(1) != "b128"
                    pending.update({r: t for r in range(int(rd.group(2)), int(rd.group(3)) + 1)})
                elif t.startswith("v_mfma"):
                    for r in regs:
                        pending.pop(r, None)
                elif not in_asm:
                    assert not regs & set(pending), (name, "register of an in-flight fragment read touched", t)
            assert not pending, (name, "fragment reads that no MFMA takes", pending)
            assert int(re.search(re.escape(name) + r"\.num_vgpr, (\d+)", text).group(1)) <= 256
            assert int(re.search(re.escape(name) + r"\.private_seg_size, (\d+)", text).group(1)) == 0
    assert seen >= 16 and transposing > 0


def test_weights_with_overlapping_rows_are_refused_by_name(no_device_check):
    x, w, one = torch.zeros(4, 64, dtype=BF), torch.zeros(16, 64, dtype=BF), torch.zeros(1, 64, dtype=BF).expand(16, 64)
    near = torch.zeros(16 * 63 + 64, dtype=BF).as_strided((16, 64), (63, 1))
    g = torch.zeros(4, 16, dtype=BF)
    x8, w8, s4, s16 = torch.zeros(4, 128, dtype=ops.FP8), torch.zeros(16, 128, dtype=ops.FP8), torch.ones(4), torch.ones(16)
    one8 = w8[:1].expand(16, 128)
    for call, name in ((lambda: ops.gated_ff(x, one, w), "w_gate"), (lambda: ops.gated_ff(x, w, near), "w_up"),
                       (lambda: ops.gated_ff_fp8(x8, s4, one8, s16, w8, s16), "w_gate"),
                       (lambda: ops.gated_ff_backward(g, x, w, one, g, g), "w_up"),
                       (lambda: ops.gated_ff_backward(g, x, near, w, g, g), "w_gate")):
        with pytest.raises(ValueError, match=name + ": rows of .* overlap"):
            call()


def test_the_library_refuses_weights_with_overlapping_rows():
    L, p, F, K = fplib.load(), 1 << 20, 16, 128
    for ld in (0, K - 1):
        assert L.fp_gated_ff_bf16(p, K, p, ld, p, K, None, None, p, F, None, None, 0, 4, F, K, 0, None, 0, None) == 1
        assert L.fp_gated_ff_backward_bf16(p, F, p, K, p, K, p, ld, p, F, p, F, p, p, None, 4, F, K, 0, p, 1 << 30, None) == 1
