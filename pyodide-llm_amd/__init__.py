"""pyodide-llm's quantized forward path on MI355X: HIP kernels for gfx950 behind the interface public/forward.js gives
its Python caller. The directory's name is not a Python identifier: load it through importlib under the name
pyodide_llm_amd (importlib.util.spec_from_file_location with submodule_search_locations=[this directory])."""
from .hip_engine import (CACHE_BLOCK, CACHE_RECENT, KINDS, KV_EIGHT, HeConfig, HeTensor, HipError, HkCache, HkPages, TensorArray, TENSORS, T, Engine, External,
                         cache_shapes, config, external, group_size, library, open_config, open_synthetic, pages_shapes, places, plan_to_config,
                         quantize_four, rope_tables, start)

__all__ = ["KINDS", "group_size", "places", "rope_tables", "HeConfig", "HeTensor", "HipError", "TensorArray", "TENSORS", "T", "Engine", "External", "config",
           "external", "library", "CACHE_BLOCK", "CACHE_RECENT", "KV_EIGHT", "HkCache", "HkPages", "cache_shapes", "pages_shapes", "quantize_four", "open_config", "open_synthetic", "plan_to_config", "start"]
