"""siliconfer_b200 -- siliconfer's Q4Linear int4 path on NVIDIA B200 (sm_100a).

Public surface:
  siliconfer_b200.kernels.cuda   -- mirror of siliconfer.kernels.neon
  siliconfer_b200.q4_linear      -- Q4Linear (torch.nn.Module)
  siliconfer_b200.q4_loader      -- _pack_and_replace_linears
  siliconfer_b200.quant          -- packers (host and device)
  siliconfer_b200.tensor_parallel-- column/row-parallel Q4Linear over NCCL
  siliconfer_b200.norm           -- RMS norm with residual, e4m3 rows with scales
  siliconfer_b200.fp8_linear     -- linear layers over e4m3 blocks (Fp8Linear)
  siliconfer_b200.rotary         -- rotary positions and their tables
  siliconfer_b200.paged_kv       -- paged e4m3 cache: append, attention (PagedKVCache)
  siliconfer_b200.attention_block-- these four as the attention half of a decoder layer
The compute lives in libsf_q4.so (C ABI: include/sf_q4.h).
"""
__version__ = "0.1.0"
