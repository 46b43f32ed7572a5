"""powershard_amd -- MI355X (gfx950) native quantized linear path of ComfyUI-PowerShard.

Modules (the first three mirror the reference modules of the same name):
  quant_linear   QuantLinear / QuantPlan / pack / unpack / install_quant_linears / build_bytes
  quant_formats  comfy_quant metadata, packed shapes, vocabulary, dequantize_module
  operations     regular_hadamard / dequantize_rows / Int8Linear / install_int8
  quant_tensor   QuantizedWeight and its three layouts (int8 rows + ConvRot, fp8 e4m3fn, uint4 groups)
  mlp            chunked Linear -> GELU(tanh) -> Linear (the Wan FFN) with the GELU in the GEMM epilogue
  norm           RMSNorm whose rows go to the quantized linears as codes
  kv_cache       PagedKVCache: a paged key-value cache in 16 bits, int8 or e4m3
  decoder        DecoderLayer: a text decoder layer on the linears, the norm and the cache
  ops            torch-facing wrappers of the HIP kernels in libpsquant.so (the decoder operators' shortest
                 host calls are in psq_direct.so, csrc/direct.cpp)
"""
__version__ = "0.1.0"
