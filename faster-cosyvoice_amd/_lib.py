"""ctypes bindings of libfcvdit.so (declared in include/fcv_dit.h, fcv_flow.h, fcv_hift.h, fcv_lm.h
and fcv_fp4.h).

The library is the only compute path: if it is missing, importing the estimator raises,
there is no fallback.  Error codes map to the exceptions the reference raises for the same
conditions (flashinfer_dit.py:326-327 ValueError for bad inputs, :235-236 and :979-983
RuntimeError for state errors).
"""

from __future__ import annotations

import ctypes
from ctypes import POINTER, c_float, c_int32, c_int64, c_size_t, c_void_p
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libfcvdit.so"

FCV_OK, FCV_ERR_INVALID, FCV_ERR_RUNTIME, FCV_ERR_STATE = 0, 1, 2, 3
FCV_MASK_FULL, FCV_MASK_CHUNK_CAUSAL = 0, 1

DIM_FIELDS = ("dim", "depth", "heads", "dim_head", "ff_dim", "mel_dim", "conv_kernel",
              "conv_groups", "rope_dim", "max_pos")

WEIGHT_FIELDS = (
    "temb_w1", "temb_b1", "temb_w2", "temb_b2", "ada_w", "ada_b", "in_w", "in_b",
    "conv1_w", "conv1_b", "conv2_w", "conv2_b", "qkv_w", "qkv_b", "out_w", "out_b",
    "ff1_w", "ff1_b", "ff2_w", "ff2_b", "proj_w", "proj_b", "rope_cos", "rope_sin",
)


class FcvDitDims(ctypes.Structure):
    _fields_ = [(name, c_int32) for name in DIM_FIELDS]


class FcvDitWeights(ctypes.Structure):
    _fields_ = [(name, c_void_p) for name in WEIGHT_FIELDS]


FLOW_MAX_DOCS = 256  # FCV_FLOW_MAX_DOCS
FLOW_DIM_FIELDS = ("vocab", "feat_dim", "channels", "lookahead", "token_mel_ratio", "spk_dim")
FLOW_WEIGHT_FIELDS = ("embed", "la1_w", "la1_b", "la2_w", "la2_b", "spk_w", "spk_b")


class FcvFlowDims(ctypes.Structure):
    _fields_ = [(name, c_int32) for name in FLOW_DIM_FIELDS]


class FcvFlowWeights(ctypes.Structure):
    _fields_ = [(name, c_void_p) for name in FLOW_WEIGHT_FIELDS]


HIFT_MAX = 4          # FCV_HIFT_MAX
HIFT_MAX_DOCS = 256   # FCV_HIFT_MAX_DOCS
_I4 = c_int32 * HIFT_MAX


class FcvHiftDims(ctypes.Structure):
    _fields_ = [
        ("in_channels", c_int32), ("base_channels", c_int32), ("nb_harmonics", c_int32),
        ("sampling_rate", c_int32), ("nsf_alpha", c_float), ("nsf_sigma", c_float),
        ("nsf_voiced_threshold", c_float), ("n_stages", c_int32), ("upsample_rates", _I4),
        ("upsample_kernels", _I4), ("n_kernels", c_int32), ("resblock_kernels", _I4),
        ("n_dilations", c_int32), ("resblock_dilations", _I4 * HIFT_MAX),
        ("source_kernels", _I4), ("source_dilations", _I4 * HIFT_MAX), ("n_fft", c_int32),
        ("hop_len", c_int32), ("conv_pre_look_right", c_int32), ("f0_channels", c_int32),
        ("lrelu_slope", c_float), ("audio_limit", c_float), ("noise_samples", c_int32),
    ]


class FcvLmLinear(ctypes.Structure):
    _fields_ = ([(n, c_void_p) for n in ("x", "w", "bias", "residual", "y")]
                + [(n, c_int64) for n in ("ldx", "ldw", "ldr", "ldy")]
                + [(n, c_int32) for n in ("m", "n", "k", "dtype", "bias_dtype", "residual_dtype",
                                          "y_dtype", "activation")])


class FcvLmQkNormRope(ctypes.Structure):
    _fields_ = ([(n, c_void_p) for n in ("qkv", "positions", "cache_rows", "rope_cos", "rope_sin",
                                         "q_weight", "k_weight", "q_out", "k_cache", "v_cache")]
                + [(n, c_int64) for n in ("qkv_row", "q_row", "k_session", "k_row", "k_head",
                                          "v_session", "v_row", "v_head")]
                + [(n, c_int32) for n in ("tokens", "n_heads", "n_kv_heads", "head_dim", "rope_dim",
                                          "max_pos", "sessions", "capacity", "dtype",
                                          "weight_dtype", "interleaved")]
                + [("eps", c_float)])


class FcvLmAttention(ctypes.Structure):
    _fields_ = ([(n, c_void_p) for n in ("q", "prefix_k", "prefix_v", "k_cache", "v_cache", "cu_q",
                                         "lengths", "slots", "out", "lse")]
                + [(n, c_int64) for n in ("q_row", "q_head", "out_row", "out_head", "pk_row",
                                          "pk_head", "pv_row", "pv_head", "k_session", "k_row",
                                          "k_head", "v_session", "v_row", "v_head")]
                + [(n, c_int32) for n in ("tokens", "batch", "n_heads", "n_kv_heads", "head_dim",
                                          "prefix_len", "sessions", "capacity", "max_q",
                                          "max_length", "dtype")]
                + [("scale", c_float)])


class FcvFp4Quantize(ctypes.Structure):
    _fields_ = ([(n, c_void_p) for n in ("w", "codes", "scales")]
                + [(n, c_int64) for n in ("ldw", "ld_codes", "ld_scales")]
                + [(n, c_int32) for n in ("n", "k", "dtype")])


class FcvFp4Linear(ctypes.Structure):
    _fields_ = ([(n, c_void_p) for n in ("x", "codes", "scales", "bias", "residual", "y")]
                + [(n, c_int64) for n in ("ldx", "ld_codes", "ld_scales", "ldr", "ldy")]
                + [(n, c_int32) for n in ("m", "n", "k", "dtype", "bias_dtype", "residual_dtype",
                                          "y_dtype", "activation")])


class FcvFp4Append(ctypes.Structure):
    _fields_ = ([(n, c_void_p) for n in ("qkv", "positions", "cache_rows", "rope_cos", "rope_sin",
                                         "q_weight", "k_weight", "q_out", "pages")]
                + [(n, c_int64) for n in ("qkv_row", "q_row", "page_stride", "head_stride")]
                + [(n, c_int32) for n in ("tokens", "n_heads", "n_kv_heads", "head_dim", "rope_dim",
                                          "max_pos", "n_pages", "dtype", "weight_dtype",
                                          "interleaved")]
                + [("eps", c_float)])


class FcvFp4Read(ctypes.Structure):
    _fields_ = ([(n, c_void_p) for n in ("pages", "rows", "k", "v")]
                + [(n, c_int64) for n in ("page_stride", "head_stride", "k_row", "v_row")]
                + [(n, c_int32) for n in ("tokens", "n_kv_heads", "head_dim", "n_pages", "dtype")])


class FcvFp4Attention(ctypes.Structure):
    _fields_ = ([(n, c_void_p) for n in ("q", "pages", "table", "lengths", "cu_q", "out", "lse")]
                + [(n, c_int64) for n in ("q_row", "q_head", "out_row", "out_head", "page_stride",
                                          "head_stride", "table_row")]
                + [(n, c_int32) for n in ("tokens", "batch", "n_heads", "n_kv_heads", "head_dim",
                                          "n_pages", "max_pages", "max_q", "max_length", "dtype")]
                + [("scale", c_float)])


# (name, restype, argtypes) of every exported entry point
SIGNATURES = {
    "fcv_last_error": (ctypes.c_char_p, []),
    "fcv_dit_create": (c_int32, [POINTER(FcvDitDims), POINTER(FcvDitWeights), POINTER(c_void_p)]),
    "fcv_dit_destroy": (c_int32, [c_void_p]),
    "fcv_dit_workspace_bytes": (c_size_t, [c_void_p, c_int32, c_int32]),
    "fcv_dit_plan": (c_int32, [c_void_p, POINTER(c_int32), c_int32, c_int32, c_int32, c_void_p,
                               c_size_t, c_void_p]),
    "fcv_dit_plan_capacity": (c_int32, [c_void_p, POINTER(c_int32), c_int32, c_int32, c_int32,
                                        c_int32, c_int32, c_void_p, c_size_t, c_void_p]),
    "fcv_dit_graph_stats": (c_int32, [c_void_p, POINTER(c_int32), POINTER(c_int32)]),
    "fcv_dit_plan_info": (c_int32, [c_void_p, POINTER(c_int32), POINTER(c_int32),
                                    POINTER(c_int32)]),
    "fcv_dit_forward": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                  c_int32, c_void_p, c_void_p]),
    "fcv_euler_cfg_step": (c_int32, [c_void_p, c_void_p, c_void_p, c_float, c_float, c_void_p]),
    "fcv_dit_solve": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                POINTER(c_float), POINTER(c_float), c_int32, c_float, c_int32,
                                c_void_p]),
    "fcv_dit_schedule_bytes": (c_size_t, [c_void_p, c_int32]),
    "fcv_dit_schedule": (c_int32, [c_void_p, POINTER(c_float), c_int32, c_void_p, c_size_t,
                                   c_void_p]),
    "fcv_dit_solve_scheduled": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                          POINTER(c_float), c_int32, c_float, c_void_p,
                                          c_size_t, c_int32, c_void_p]),
    "fcv_pack_padded": (c_int32, [c_void_p, c_void_p, c_int32, c_int32, c_int32, c_void_p,
                                  c_void_p]),
    "fcv_unpack_padded": (c_int32, [c_void_p, c_void_p, c_int32, c_int32, c_int32, c_void_p,
                                    c_void_p]),
    "fcv_dit_probe_arm": (c_int32, [c_void_p, c_int32, c_int32, c_int32]),
    "fcv_dit_probe_read": (c_int32, [c_void_p, POINTER(c_float), c_int32, POINTER(c_int32)]),
    # include/fcv_flow.h
    "fcv_flow_workspace_bytes": (c_size_t, [POINTER(FcvFlowDims), c_int32]),
    "fcv_flow_token_features": (c_int32, [POINTER(FcvFlowDims), POINTER(FcvFlowWeights), c_void_p,
                                          POINTER(c_int32), POINTER(c_int32), c_int32, c_void_p,
                                          c_void_p, c_size_t, c_void_p]),
    "fcv_flow_token_features_noalloc": (c_int32, [POINTER(FcvFlowDims), POINTER(FcvFlowWeights),
                                                  c_void_p, POINTER(c_int32), POINTER(c_int32),
                                                  c_int32, c_void_p, c_void_p]),
    "fcv_flow_speaker": (c_int32, [POINTER(FcvFlowDims), POINTER(FcvFlowWeights), c_void_p,
                                   c_int32, c_void_p, c_void_p]),
    "fcv_flow_prompt_cond": (c_int32, [POINTER(FcvFlowDims), c_void_p, POINTER(c_int32),
                                       POINTER(c_int32), c_int32, c_void_p, c_void_p]),
    # include/fcv_hift.h
    "fcv_hift_weight_count": (c_int32, [POINTER(FcvHiftDims)]),
    "fcv_hift_create": (c_int32, [POINTER(FcvHiftDims), POINTER(c_void_p), c_int32,
                                  POINTER(c_void_p)]),
    "fcv_hift_destroy": (c_int32, [c_void_p]),
    "fcv_hift_packed_bytes": (c_size_t, [c_void_p]),
    "fcv_hift_pack_weights": (c_int32, [c_void_p, c_void_p, c_size_t, c_void_p]),
    "fcv_hift_use_packed": (c_int32, [c_void_p, c_void_p, c_size_t]),
    "fcv_hift_weight_packed": (c_int32, [c_void_p, c_int32]),
    "fcv_hift_output_samples": (ctypes.c_int64, [c_void_p, c_int32, c_int32]),
    "fcv_hift_workspace_bytes": (c_size_t, [c_void_p, POINTER(c_int32), POINTER(c_int32),
                                            c_int32]),
    "fcv_hift_inference": (c_int32, [c_void_p, c_void_p, POINTER(c_int32), POINTER(c_int32),
                                     c_int32, c_void_p, c_void_p, c_void_p, c_size_t,
                                     c_void_p]),
    "fcv_hift_workspace_bytes_capacity": (c_size_t, [c_void_p, c_int32, c_int32]),
    "fcv_hift_inference_capacity": (c_int32, [c_void_p, c_void_p, POINTER(c_int32),
                                              POINTER(c_int32), c_int32, c_int32, c_int32,
                                              c_void_p, c_void_p, c_void_p, c_size_t, c_int32,
                                              c_void_p]),
    "fcv_hift_graph_stats": (c_int32, [c_void_p, POINTER(c_int32), POINTER(c_int32)]),
    # include/fcv_lm.h
    "fcv_lm_linear_workspace_bytes": (c_size_t, [POINTER(FcvLmLinear)]),
    "fcv_lm_linear": (c_int32, [POINTER(FcvLmLinear), c_void_p, c_size_t, c_void_p]),
    "fcv_lm_linear_plan": (c_int32, [POINTER(FcvLmLinear), POINTER(c_int32), POINTER(c_int32)]),
    "fcv_lm_qk_norm_rope": (c_int32, [POINTER(FcvLmQkNormRope), c_void_p]),
    "fcv_lm_prefix_attention_workspace_bytes": (c_size_t, [POINTER(FcvLmAttention)]),
    "fcv_lm_prefix_attention": (c_int32, [POINTER(FcvLmAttention), c_void_p, c_size_t, c_void_p]),
    # include/fcv_fp4.h
    "fcv_fp4_quantize": (c_int32, [POINTER(FcvFp4Quantize), c_void_p]),
    "fcv_fp4_linear_workspace_bytes": (c_size_t, [POINTER(FcvFp4Linear)]),
    "fcv_fp4_linear": (c_int32, [POINTER(FcvFp4Linear), c_void_p, c_size_t, c_void_p]),
    "fcv_fp4_linear_plan": (c_int32, [POINTER(FcvFp4Linear), POINTER(c_int32), POINTER(c_int32)]),
    "fcv_fp4_page_bytes": (c_size_t, [c_int32]),
    "fcv_fp4_append": (c_int32, [POINTER(FcvFp4Append), c_void_p]),
    "fcv_fp4_read": (c_int32, [POINTER(FcvFp4Read), c_void_p]),
    "fcv_fp4_attention_workspace_bytes": (c_size_t, [POINTER(FcvFp4Attention)]),
    "fcv_fp4_attention_plan": (c_int32, [POINTER(FcvFp4Attention)] + [POINTER(c_int32)] * 4),
    "fcv_fp4_attention": (c_int32, [POINTER(FcvFp4Attention), c_void_p, c_size_t, c_void_p]),
    "fcv_copy_pages": (c_int32, [c_void_p, c_int32, c_int64, c_int32, c_int64, c_int64,
                                 c_void_p, c_void_p, c_int32, c_void_p]),
}

STAGES = ("qkv", "attention", "out_proj", "ff1", "ff2", "ln_mod", "conv", "adaln", "in_proj",
          "proj_out", "euler", "forward")

_LIB: ctypes.CDLL | None = None


def load() -> ctypes.CDLL:
    """Load libfcvdit.so once; raise ImportError when it has not been built."""
    global _LIB
    if _LIB is not None:
        return _LIB
    if not LIB_PATH.exists():
        raise ImportError(f"{LIB_PATH} is missing: build it with `python faster-cosyvoice_amd/build.py` "
                          "(the HIP library is the only compute path)")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, (restype, argtypes) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    _LIB = lib
    return lib


def check(rc: int) -> None:
    """Raise the Python exception that matches a library status code."""
    if rc == FCV_OK:
        return
    msg = load().fcv_last_error().decode(errors="replace")
    if rc == FCV_ERR_INVALID:
        raise ValueError(msg)
    raise RuntimeError(msg)
