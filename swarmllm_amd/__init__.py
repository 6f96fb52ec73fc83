"""swarmllm_amd — SwarmLLM's quantized matmul path (candle QTensor / QMatMul
over GGUF Q8_0, Q4_K, Q6_K, IQ4_NL, MXFP4) as hand-written HIP kernels for
AMD Instinct MI355X (gfx950), with the steps of a decoder layer between its
products (norm into a quantized activation, a paged Q8_0 cache, the attention
over it) and what a batch of many requests needs around them (page tables on
the device, low-rank adapters, sampling), behind the C ABI of include/qmm.h."""

from ._lib import QmmError, lib  # noqa: F401
from .batch import BatchRows, PageTables  # noqa: F401
from .kvcache import KvCache  # noqa: F401
from .lora import Adapters  # noqa: F401
from .norm import NormOut, rms_norm_act  # noqa: F401
from .qtensor import (MOE_CARD_ONE_ROW_MAX_TOKENS, GgmlDType, QAct, QMatMul, QTensor, fill_normal,  # noqa: F401
                      forward_glu, glu, mmq_few_rows_line, moe_forward, moe_prompt_on_tensor_cores,
                      moe_uses_prompt_kernel, prepare, prepared, set_force_dmmv)
from .sampling import Sampled, sample  # noqa: F401

__all__ = ["MOE_CARD_ONE_ROW_MAX_TOKENS", "Adapters", "BatchRows", "GgmlDType", "KvCache", "NormOut", "PageTables",
           "QAct", "QMatMul", "QTensor", "QmmError", "Sampled", "fill_normal", "forward_glu", "glu", "lib",
           "mmq_few_rows_line", "moe_forward", "moe_prompt_on_tensor_cores", "moe_uses_prompt_kernel", "prepare",
           "prepared", "rms_norm_act", "sample", "set_force_dmmv"]
