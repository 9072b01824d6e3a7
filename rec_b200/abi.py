"""ctypes mirror of include/rec_b200.h (structures and constants)."""
from __future__ import annotations

import ctypes as C

REC_OK = 0
REC_EINVAL = -1
REC_ECUDA = -2
REC_ESTATE = -3
REC_ELIMIT = -4
REC_DEV_BULK_TIMEOUT = 1
REC_DEV_COUNTER_TIMEOUT = 2
REC_DEV_BAD_TOKEN = 3
REC_DEV_BAD_POSITION = 4
REC_DEV_BAD_PAGE = 5

REC_SCALE_FP16 = 0
REC_SCALE_BF16 = 1
REC_ROUTER_SOFTMAX = 0
REC_ROUTER_SIGMOID = 1
REC_FLAG_SINKS = 1
REC_FLAG_QK_NORM = 2
# layer kinds (RecLayerWeights.kind bits)
REC_LAYER_DENSE = 1
REC_LAYER_NO_ROPE = 2
REC_LAYER_SLIDING = 4
# element types of the batched-decode operators
REC_T_BF16 = 0
REC_T_FP16 = 1
REC_T_FP32 = 2


class RecModelDesc(C.Structure):
    _fields_ = [
        ("hidden", C.c_int32),
        ("n_layers", C.c_int32),
        ("n_q_heads", C.c_int32),
        ("n_kv_heads", C.c_int32),
        ("head_dim", C.c_int32),
        ("n_experts", C.c_int32),
        ("top_k", C.c_int32),
        ("moe_inter", C.c_int32),
        ("vocab", C.c_int32),
        ("group_size", C.c_int32),
        ("scale_dtype", C.c_int32),
        ("kv_bits", C.c_int32),
        ("router_mode", C.c_int32),
        ("flags", C.c_int32),
        ("rms_eps", C.c_float),
        ("rope_theta", C.c_float),
        ("shared_inter", C.c_int32),
        ("dense_inter", C.c_int32),
        ("sliding_window", C.c_int32),
        ("embed_bits", C.c_int32),
        ("kv_value_bits", C.c_int32),
    ]


class RecQMat(C.Structure):
    _fields_ = [("w", C.c_void_p), ("scales", C.c_void_p), ("biases", C.c_void_p)]


class RecLayerWeights(C.Structure):
    _fields_ = [
        ("input_norm", C.c_void_p),
        ("post_norm", C.c_void_p),
        ("q", RecQMat),
        ("k", RecQMat),
        ("v", RecQMat),
        ("o", RecQMat),
        ("router", C.c_void_p),
        ("expert_bias", C.c_void_p),
        ("gate", RecQMat),
        ("up", RecQMat),
        ("down", RecQMat),
        ("sinks", C.c_void_p),
        ("q_norm", C.c_void_p),
        ("k_norm", C.c_void_p),
        ("kind", C.c_int32),
        ("shared_gate", RecQMat),
        ("shared_up", RecQMat),
        ("shared_down", RecQMat),
    ]


class RecGlobalWeights(C.Structure):
    _fields_ = [("embed", RecQMat), ("final_norm", C.c_void_p), ("lm_head", RecQMat)]


class RecKVLayer(C.Structure):
    _fields_ = [
        ("k_codes", C.c_void_p),
        ("k_scales", C.c_void_p),
        ("k_biases", C.c_void_p),
        ("v_codes", C.c_void_p),
        ("v_scales", C.c_void_p),
        ("v_biases", C.c_void_p),
    ]


class RecSampling(C.Structure):
    _fields_ = [
        ("temperature", C.c_float),
        ("top_k", C.c_int32),
        ("top_p", C.c_float),
        ("repetition_penalty", C.c_float),
        ("presence_penalty", C.c_float),
    ]


class RecShard(C.Structure):
    _fields_ = [
        ("world", C.c_int32),
        ("rank", C.c_int32),
        ("expert_lo", C.c_int32),
        ("expert_hi", C.c_int32),
        ("super_lo", C.c_int32),
        ("super_hi", C.c_int32),
        ("capacity_total", C.c_int32),
        ("exchange", C.c_void_p * 8),
        ("schedule", C.c_int32),
    ]


class RecPagedKV(C.Structure):
    _fields_ = [
        ("k", C.c_void_p),
        ("v", C.c_void_p),
        ("k_scales", C.c_void_p),
        ("k_biases", C.c_void_p),
        ("v_scales", C.c_void_p),
        ("v_biases", C.c_void_p),
        ("k_stride", C.c_int64 * 3),
        ("v_stride", C.c_int64 * 3),
        ("k_scale_stride", C.c_int64 * 3),
        ("v_scale_stride", C.c_int64 * 3),
        ("n_pages", C.c_int32),
        ("page_size", C.c_int32),
        ("n_kv_heads", C.c_int32),
        ("head_dim", C.c_int32),
        ("k_bits", C.c_int32),
        ("v_bits", C.c_int32),
        ("dtype", C.c_int32),
    ]


class RecPagedTable(C.Structure):
    _fields_ = [
        ("table", C.c_void_p),
        ("table_stride", C.c_int64),
        ("width", C.c_int32),
        ("batch", C.c_int32),
    ]


class RecPagedAttn(C.Structure):
    _fields_ = [
        ("q", C.c_void_p),
        ("q_batch_stride", C.c_int64),
        ("q_head_stride", C.c_int64),
        ("out", C.c_void_p),
        ("out_batch_stride", C.c_int64),
        ("out_head_stride", C.c_int64),
        ("lse", C.c_void_p),
        ("lengths", C.c_void_p),
        ("sinks", C.c_void_p),
        ("n_q_heads", C.c_int32),
        ("scale", C.c_float),
        ("softcap", C.c_float),
        ("window", C.c_int32),
        ("weights_in", C.c_void_p),
        ("weights_out", C.c_void_p),
        ("decay", C.c_float),
    ]


class RecPagedEvict(C.Structure):
    _fields_ = [
        ("lengths", C.c_void_p),
        ("lengths_out", C.c_void_p),
        ("budget", C.c_int32),
        ("weights_in", C.c_void_p),
        ("weights_out", C.c_void_p),
        ("positions_in", C.c_void_p),
        ("positions_out", C.c_void_p),
        ("keep_from", C.c_void_p),
        ("keep_below", C.c_int32),
    ]


class RecLogitRules(C.Structure):
    _fields_ = [
        ("history", C.c_void_p),
        ("history_cap", C.c_int32),
        ("history_len", C.c_void_p),
        ("prompt_len", C.c_void_p),
        ("repetition", C.c_void_p),
        ("frequency", C.c_void_p),
        ("presence", C.c_void_p),
        ("bias_ids", C.c_void_p),
        ("bias_values", C.c_void_p),
        ("n_bias", C.c_int32),
        ("allow", C.c_void_p),
        ("allow_stride", C.c_int64),
    ]
