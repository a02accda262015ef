"""What the 16- and 32-bit products write, and that they write nothing else.

A TMA store cuts a box off at the tensor's last column in whole pieces of 16 bytes, so where a row of C is no multiple of that the
columns between n and the leading dimension are at stake; a caller may keep values of his own there."""

import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class GemmArgs(C.Structure):
    _fields_ = [("arith", C.c_int), ("m", C.c_int), ("n", C.c_int), ("k", C.c_int), ("a", C.c_void_p), ("b", C.c_void_p),
                ("lda", C.c_longlong), ("ldb", C.c_longlong), ("b_transposed", C.c_int), ("c", C.c_void_p), ("ldc", C.c_longlong),
                ("c16", C.c_void_p), ("c16_kind", C.c_int), ("ldc16", C.c_longlong), ("splits", C.c_int), ("workspace", C.c_void_p),
                ("function", C.c_void_p), ("reduce_function", C.c_void_p), ("epilogue_inputs", C.c_void_p * 6),
                ("num_epilogue_inputs", C.c_int), ("status", C.c_void_p), ("variant", C.c_int), ("tile_n", C.c_int), ("has_epilogue", C.c_int)]


@pytest.mark.parametrize("arith, half", [(2, "bf16"), (3, "f16"), (1, None)])
@pytest.mark.parametrize("outputs", ("c", "c16", "both"))
@pytest.mark.parametrize("m, n, pad", [(512, 516, 8), (300, 513, 8), (600, 1027, 16), (257, 290, 32), (512, 520, 8)])
@pytest.mark.parametrize("variant", (8 | 32, 8 | 16, 0))
def test_only_c_is_written(mc, arith, half, outputs, m, n, pad, variant):
    """Variant bit 8 takes the SM-pair kernel, with bit 16 its two-tile form. The operands are whole numbers of few bits: sums are exact."""
    import torch

    torch.manual_seed(n)
    k = 72
    a = torch.randint(-4, 5, (m, k)).double()
    b = torch.randint(-4, 5, (n, k)).double()
    want = (a @ b.T).numpy()
    t = {"bf16": torch.bfloat16, "f16": torch.float16, None: torch.float32}[half]
    ta, tb = a.to(t).cuda(), b.to(t).cuda()
    half_t, half_kind = (torch.float16, 2) if half == "f16" else (torch.bfloat16, 1)
    ldc = (n + pad + 7) // 8 * 8
    c = torch.full((m + 1, ldc), 7.0, device="cuda")
    c16 = torch.full((m + 1, ldc), 7.0, device="cuda", dtype=half_t)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    args = GemmArgs(arith=arith, m=m, n=n, k=k, a=ta.data_ptr(), b=tb.data_ptr(), lda=k, ldb=k, b_transposed=1, splits=1, variant=variant,
                    status=status.data_ptr(), c16_kind=half_kind, ldc=ldc, ldc16=ldc)
    if outputs != "c16":
        args.c = c.data_ptr()
    if outputs != "c":
        args.c16 = c16.data_ptr()
    torch.cuda.synchronize()
    lib = mc.lib()
    lib.mcd_gemm.restype = C.c_int
    assert lib.mcd_gemm(C.byref(args), C.c_void_p(0)) == 0, lib.mcd_last_error()
    torch.cuda.synchronize()
    assert status.item() == 0
    for out, asked, tt in ((c, outputs != "c16", torch.float32), (c16, outputs != "c", half_t)):
        assert (out[m] == 7).all() and (out[:, n:] == 7).all()
        if asked:
            assert np.array_equal(out[:m, :n].double().cpu().numpy(), torch.from_numpy(want).to(torch.float32).to(tt).double().numpy())
        else:
            assert (out == 7).all()



@pytest.mark.parametrize("arith, half", [(2, "bf16"), (3, "f16"), (1, None)])
@pytest.mark.parametrize("m, n, k", [(300, 300, 70), (64, 130, 1001), (512, 512, 129), (1, 300, 67)])
def test_what_lies_behind_the_rows_of_the_operands_is_not_read(mc, arith, half, m, n, k):
    """NaN between k and the leading dimension of both operands, in every form of the kernels."""
    import torch

    torch.manual_seed(k)
    a, b = torch.randint(-4, 5, (m, k)).double(), torch.randint(-4, 5, (n, k)).double()
    t = {"bf16": torch.bfloat16, "f16": torch.float16, None: torch.float32}[half]
    ld = (k + 15) // 8 * 8
    pads = [torch.full((rows, ld), float("nan"), dtype=t, device="cuda") for rows in (m, n)]
    pads[0][:, :k], pads[1][:, :k] = a.to(t).cuda(), b.to(t).cuda()
    want = (a @ b.T).numpy()
    lib = mc.lib()
    lib.mcd_gemm.restype = C.c_int
    for variant, splits in ((0, 1), (4, 1), (8 | 32, 1), (8 | 16, 1), (0, 2), (64, 2)):
        c = torch.full((m, n), 7.0, device="cuda")
        ws = torch.empty(splits * m * n, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        args = GemmArgs(arith=arith, m=m, n=n, k=k, a=pads[0].data_ptr(), b=pads[1].data_ptr(), lda=ld, ldb=ld, b_transposed=1, splits=splits,
                        variant=variant, status=status.data_ptr(), c=c.data_ptr(), ldc=n, workspace=ws.data_ptr())
        torch.cuda.synchronize()
        assert lib.mcd_gemm(C.byref(args), C.c_void_p(0)) == 0, lib.mcd_last_error()
        torch.cuda.synchronize()
        assert status.item() == 0
        assert np.array_equal(c.double().cpu().numpy(), want), (variant, splits)
