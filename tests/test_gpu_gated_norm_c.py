"""The C entries of gated_add_rms_norm on calls that the tensor entry point does not make."""
import ctypes

import pytest
import torch

import blockcheck as bc
import decaycheck as dc
from lfcheck import TORCH_DT, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate_rows", [0, 1, 4, 12])
def test_no_gate_with_gate_rows(gpu, dtype, post, gate_rows):
    """A NULL gate is 1 whatever the description says of gate rows: nothing is read through it, forward or backward."""
    import laplacianformer_amd as lf
    import laplacianformer_amd._lib as L

    lib, t, rows, scale, eps = lf.capi(), TORCH_DT[dtype], 12, 0.5, 1e-5
    code, p = lf.dtype_code(t), lambda a: None if a is None else ctypes.c_void_p(a.data_ptr())
    for W in (8, 333, 1000, 4100):
        print(f"gated norm, no gate, gate_rows {gate_rows} {dtype} {post} {W}", flush=True)
        x, res, gy, gs = (gen((rows, W), 20 + i, dtype) for i in range(4))
        w, wp = gen((W,), 24, dtype), gen((W,), 25, dtype) if post else None
        ref = dc.gated_norm(x, w, res, wp, None, scale, eps, gy, gs)
        X, R, GY, GS, Wd, P = (None if a is None else a.to(gpu) for a in (x, res, gy, gs, w, wp))
        y, total, dx, dr = (torch.empty(rows, W, dtype=t, device=gpu) for _ in range(4))
        dw, dwp = (torch.empty(W, dtype=t, device=gpu) for _ in range(2))
        rstd, rpost = (torch.empty(rows, dtype=torch.float32, device=gpu) for _ in range(2))
        d = L.GatedNorm(rows=rows, width=W, x_stride=W, residual_stride=W, gate_rows=gate_rows, gate_stride=W, weight_dtype=code,
                        post_weight_dtype=code, gate_dtype=code, scale=scale, eps=eps)
        st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        lf.check(lib.lfamd_gated_add_rms_norm(code, ctypes.byref(d), p(X), p(R), p(Wd), p(P), None, p(y), p(total), p(rstd),
                                              p(rpost) if post else None, st))
        need = lib.lfamd_gated_add_rms_norm_backward_workspace_size(code, ctypes.byref(d))
        ws = torch.empty(need // 4, dtype=torch.float32, device=gpu)
        lf.check(lib.lfamd_gated_add_rms_norm_backward(code, ctypes.byref(d), p(GY), W, p(GS), W, p(X), p(R), p(Wd), p(P), None, p(rstd),
                                                       p(rpost) if post else None, p(dx), p(dr), p(dw), p(dwp) if post else None, None,
                                                       p(ws), need, st))
        got = {"y": y, "sum": total, "dx": dx, "dres": dr, "dw": dw, **({"dwp": dwp} if post else {})}
        for name, a in got.items():
            bc.assert_within(a, *ref[name], (dtype, post, gate_rows, W, name))
