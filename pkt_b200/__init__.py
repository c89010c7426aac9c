"""pkt_b200: B200-native (sm_100a) persistent training megakernel with pkt's host API.

Everything here calls libpkt_b200.so through its C-ABI (include/pkt_b200.h).
"""
from ._lib import PktError, load as _load  # noqa: F401
from .runtime import (AxpyArgs, GemmDesc, LinearBackwardArgs, LinearForwardArgs, MSELossArgs,  # noqa: F401
                      OpCode, Runtime, SGDUpdateArgs, Task, ZeroMemoryArgs, axpy, decode_args,
                      encode_args, make_tasks)
from .ops import (DTYPE_BF16, DTYPE_E4M3, DTYPE_E5M2, DTYPE_F32, AdamW, AdamWTensor, Fp8GemmDesc,  # noqa: F401
                  Fp8QuantizeDesc, LayerNormDesc, fp8_gemm, ops_status, fp8_quantize,
                  layernorm_backward, layernorm_backward_workspace, layernorm_forward)
from .mlp import MLP, from_bf16_bits, to_bf16_bits  # noqa: F401

_load()
