"""The outputs that the C interface allows to be inputs: a layer's output in its residual's place, the norm
step's hidden in its residual's or features' place and its normed in its features'. The bits are those of
separate outputs."""
import pytest
import torch

from sparseconv import _native

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# CUDA cores, W resident and streamed, pairs of CTAs, copies into whole rows
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,Ci,Co", [(1, 8, 8), (333, 35, 13), (50003, 64, 256), (200001, 64, 16), (3001, 1024, 256),
                                     (20011, 512, 520), (20001, 257, 131)])
def test_linear_into_its_residual(M, Ci, Co, dtype, act):
    if dtype == "fp32":
        M = min(M, 4001)
    g = torch.Generator(device="cuda").manual_seed(M)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(DT[dtype])
    x, w, b, r = mk(M, Ci), mk(Co, Ci), mk(Co), mk(M, Co)
    want, want_z = _native.linear_forward(x, w, b, r, act, keep_preact=True)
    lib, z, code = _native.load_library(), torch.empty_like(r), _native.DTYPE_CODES[DT[dtype]]
    need = lib.spconv_linear_forward_workspace_bytes(code, M, Ci, Co, 1, 1)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
    assert lib.spconv_linear_forward(
        x.data_ptr(), code, M, Ci, w.data_ptr(), b.data_ptr(), r.data_ptr(), Co, _native.ACTIVATIONS[act], r.data_ptr(),
        z.data_ptr(), ws.data_ptr(), need, 0, _native.mapped_status(0), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(r, want) and torch.equal(z, want_z)


# rows through registers, through shared memory (also with odd ends), and a block a row
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,C", [(5, 64), (700, 35), (60001, 64), (1000003, 3), (60003, 129), (40000, 256), (900, 300), (501, 2048),
                                 (77, 8192)])
@pytest.mark.parametrize("hidden,normed", [("r", None), ("x", None), (None, "x"), ("r", "x")])
def test_norm_step_into_its_inputs(M, C, dtype, hidden, normed):
    g = torch.Generator(device="cuda").manual_seed(C)
    mk = lambda *s, t=torch.float32: torch.randn(*s, generator=g, device="cuda").to(t)
    x, r = mk(M, C, t=DT[dtype]), mk(M, C, t=DT[dtype])
    ps = (mk(3, C), mk(C), mk(C), mk(C), mk(C))
    off = torch.tensor([0, M // 3, M // 2, M], dtype=torch.int32, device="cuda")
    settings = (ps, off, 0.5, "layer", "rms", 1e-5)
    want = _native.residual_norm_forward(x, r, *settings)
    a = _native._norm_args(x, r, *settings)
    out = {None: None, "x": x, "r": r}
    h, y = (torch.empty_like(x) if out[k] is None else out[k] for k in (hidden, normed))
    a.hidden, a.normed = h.data_ptr(), y.data_ptr()
    assert _native.load_library().spconv_residual_norm_forward(a, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(h, want[0]) and torch.equal(y, want[1])
