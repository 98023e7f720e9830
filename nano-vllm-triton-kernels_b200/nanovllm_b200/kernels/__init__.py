"""The B200 kernel modules, laid out as the reference's nanovllm/kernels package (qk_norm_rope_kv.py, rms_norm.py,
swiglu.py, matmul.py) plus attention.py for the attention layer's KV-cache write and decode attention, kv_quant.py for
the 8-bit KV cache and cache_attention.py for the attention of drafted trees and over that cache. The reference
picks its kernels by the string nanovllm.kernels.backend (nanovllm/kernels/__init__.py:1-5); nanovllm_b200.install()
adds "b200" to that switch."""
