"""B200-native H3 video-VAE INT8 encode/decode path (sm_100a kernels behind a C ABI).

Submodules:
  kernels   tensor-level wrappers of every C entry point (libh3vae_b200.so)
  kv_cache  paged INT8 key/value cache of one attention layer
  streaming TokenStream: the decoder blocks over a clip that arrives in pieces, on that cache
  opt       drop-in mirrors of the reference's opt/* entry points
  model     H3-structured encoder/decoder assembled from those kernels
  runtime   H3VAEPyOptRuntime (ComfyUI first_stage_model) and tile scheduling
  nodes     the H3VAEPyOptLoader ComfyUI node
"""
__version__ = "0.1.0"
