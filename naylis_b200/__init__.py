"""naylis_b200 — B200-native (sm_100a) Mixture-of-Memory hot path for Naylis.

Public surface:
  naylis_b200.mom_kernels   the dispatch door (preflight, resolve_mode, mom_read,
                            announce, and the added mom_route) for mode "sm100"
  naylis_b200.model.MoMLayer  drop-in MoM layer (reference constructor and keys)
  naylis_b200.data_parallel   explicit bucketed NCCL gradient all-reduce
  naylis_b200.attention       serving attention: packed prompts, one token over a
                            paged key-value cache, the rotary embedding with the
                            cache write, the cache itself, in bf16 or in 4 bits
  naylis_b200.scoring         token log probabilities, entropy, alternatives; which
                              drafted tokens stay
  naylis_b200.generate        answering with the decoder (generate, Session, score),
                              also with a smaller model's drafts
  naylis_b200.build           in-tree nvcc build of libnaylis_mom.so
"""
from . import mom_kernels  # noqa: F401

__all__ = ["mom_kernels"]
