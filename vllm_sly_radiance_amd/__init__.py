"""MI355X-native MXFP4 W4A8 linear-layer path (gfx950), a drop-in for the MXFP4 W4A8 path of
vllm-sly-radiance (sly/mxfp4/radiance_mxfp4.py + radiance_mxfp4_fp8.hip).

  radiance_mxfp4   custom ops radiance::mxfp4_linear[_pq] and the vLLM kernel plugin
  _native          ctypes binding of libw4a8_mxfp4.so (C ABI in include/w4a8_mxfp4.h)
  radiance_kv4     attention over a paged 4-bit key/value cache: head norm + rotation, append,
                   attention, gather, page moves (ops radiance::kv4_*, radiance::qk_norm_rope*)
  kv4_pool         the host's side of that cache: pages, forks, steps of a batch
  _native_kv4      ctypes binding of libkv4_attn.so (C ABI in include/kv4_attn.h)
  radiance_gdn     linear-attention layers between their projections: causal convolution, gated delta
                   rule (ops radiance::causal_conv, ::gated_delta_rule)
  radiance_sample  tokens from logits: temperature, top-k, top-p, min-p (op radiance::sample)
  _native_decode   ctypes binding of libdecode_ops.so (C ABI in include/decode_ops.h)
  synthetic        seeded operands with the benchmark distributions
  build            hipcc recipe for the libraries
"""
