"""Operators built on the HIP kernels: GEMM / split-K GEMM (``matmul``), the gated GEMM (``swiglu``), conv2d forward
(``conv2d``), microscaled 4-bit products (``mx``), the mixture of experts (``moe``), linear layers (``linear``), layer normalisation (``norm``)
and products grouped by expert (``grouped``)."""
import importlib

# ``ops.matmul`` names both a module and, once imported, the dispatcher it defines: bind the names explicitly
_matmul_module = importlib.import_module("tritonix_amd.ops.matmul")
_swiglu_module = importlib.import_module("tritonix_amd.ops.swiglu")
_conv2d_module = importlib.import_module("tritonix_amd.ops.conv2d")
_mx_module = importlib.import_module("tritonix_amd.ops.mx")
_moe_module = importlib.import_module("tritonix_amd.ops.moe")
_linear_module = importlib.import_module("tritonix_amd.ops.linear")
_norm_module = importlib.import_module("tritonix_amd.ops.norm")
_grouped_module = importlib.import_module("tritonix_amd.ops.grouped")

__all__ = []
for _module, _names in ((_matmul_module, ("matmul", "triton_matmul", "hip_matmul", "matmul_splitk", "matmul_kernel",
                                           "gemm_splitk_kernel")),
                        (_swiglu_module, ("glu_kernel", "swiglu_kernel", "glu", "swiglu", "swiglu_ffn", "fused_glu")),
                        (_conv2d_module, ("conv2d_forward", "conv2d_forward_kernel", "torch_conv2d_forward")),
                        (_mx_module, tuple(_mx_module.__all__)), (_moe_module, tuple(_moe_module.__all__)),
                        (_linear_module, tuple(_linear_module.__all__)), (_norm_module, tuple(_norm_module.__all__)),
                        (_grouped_module, tuple(_grouped_module.__all__))):
    for _name in _names:
        globals()[_name] = getattr(_module, _name)
        __all__.append(_name)
del _module, _names, _name
