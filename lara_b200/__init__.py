"""LARA B200: the grouped-query streaming-attention path on sm_100a.

* ``lara_b200.attn_driver`` -- drop-in for the reference host driver
  (``sw/attn_driver.py``), backed by the C-ABI context of liblara_b200.so.
* ``lara_b200.ops`` -- torch-tensor front end of the stateless kernels
  (decode, split-KV partials + LSE combine, KV append, bf16 pack, dense
  transaction, prefill).
* ``lara_b200.paged`` / ``lara_b200.kvquant`` -- paged KV caches in bf16 and in 8
  bits (int8, fp8 e4m3), with the decode that reads them; in bf16 also a decode
  behind a shared prefix, one that scores its slots, and eviction.
* ``lara_b200.workloads`` -- seeded synthetic inputs of the benchmark configs.
* ``lara_b200.build`` -- compiles liblara_b200.so (nvcc) and the _binding of
  the calls made once per layer and token, in-tree.

The library is loaded by ``lara_b200._native`` (on first use of ``lib`` /
``check`` here, or on import of any module that computes); a missing or
stale library raises there -- there is no CPU fallback.
"""

_NATIVE = ("lib", "check", "LaraError", "LaraConfigError", "LaraTimeout")

__all__ = list(_NATIVE)


def __getattr__(name):
    if name in _NATIVE:
        from . import _native

        return getattr(_native, name)
    raise AttributeError(f"module 'lara_b200' has no attribute {name!r}")
