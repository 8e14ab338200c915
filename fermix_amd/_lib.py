"""ctypes binding of the in-tree HIP library ``libfermix_amd.so`` (C ABI declared in
``include/fermix.h``). The product path has no fallback: if the library is missing the
calls raise ``FermixLibraryError``."""

import ctypes
import os

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libfermix_amd.so")

FX_OK = 0

# the prec argument (include/fermix.h): the product mode and, for the float32 slogdet /
# det entry points, option bits
FX_PREC_IEEE = 0
FX_PREC_BF16X3 = 1
FX_PREC_MASK = 0x0F
FX_LU_BLOCK_64 = 0x100
FX_LU_BLOCK_128 = 0x200

# fields of struct fx_tune, in order (int32 each; 3 reserved int32 follow)
TUNE_FIELDS = (
    "fused_max_n",
    "lu_pair_above_n",
    "lu_direct_max_n",
    "pf_block64_min_n",
    "pf_block64_max_m",
    "gemm128_min_mn",
    "gemm128_min_k",
    "gemm128_tout",
    "gemm128_x3_min_mn",
    "gemm128_x3_min_k",
    "gemm128_x3_tout",
    "f64_reg_max_n",
    "f64_strip16_max_n",
    "pf_overlap_max_half",
    "pf_overlap_min_work",
    "lu_split_min_work",
    "lu_generic_above_n",
)


class FxTune(ctypes.Structure):
    """struct fx_tune of include/fermix.h."""

    _fields_ = [(f, ctypes.c_int32) for f in TUNE_FIELDS] + [("reserved", ctypes.c_int32 * 3)]


_p = ctypes.c_void_p
_i64 = ctypes.c_int64
_i32 = ctypes.c_int32
_sz = ctypes.c_size_t

# name -> (restype, argtypes); every function declared in include/fermix.h
SIGNATURES = {
    "fx_status_string": (ctypes.c_char_p, [ctypes.c_int]),
    "fx_abi_version": (ctypes.c_int, []),
    "fx_lu_padded_size": (_i32, [_i32]),
    "fx_pf_padded_size": (_i32, [_i32]),
    "fx_tune_table": (ctypes.c_int, [ctypes.c_char_p, ctypes.POINTER(FxTune)]),
    "fx_tune_override": (ctypes.c_int, [ctypes.POINTER(FxTune)]),
    "fx_tune_active": (ctypes.c_int, [ctypes.POINTER(FxTune)]),
    "fx_slogdet_f32_workspace": (_sz, [_i64, _i32]),
    "fx_slogdet_f32": (ctypes.c_int, [_p, _i64, _i32, _p, _p, _i32, _p, _sz, _p]),
    "fx_slogdet_parts_f32_workspace": (_sz, [_i64, _i32]),
    "fx_slogdet_parts_f32": (
        ctypes.c_int,
        [_p, _i64, _i32, _i32, _p, _p, _p, _p, _p, _i32, _p, _sz, _p],
    ),
    "fx_slogdet_factors_f32_workspace": (_sz, [_i64, _i32]),
    "fx_slogdet_factors_f32": (ctypes.c_int, [_p, _i64, _i32, _p, _p, _p, _p, _i32, _p, _sz, _p]),
    "fx_slogdet_inverse_f32_workspace": (_sz, [_i64, _i32]),
    "fx_slogdet_inverse_f32": (ctypes.c_int, [_p, _p, _p, _p, _i64, _i32, _i32, _p, _i32, _p, _sz, _p]),
    "fx_slogdet_f32_noalloc": (ctypes.c_int, [_p, _i64, _i32, _p, _p, _p]),
    "fx_slogdet_f32_noalloc_batch": (_i64, [_i64, _i32]),
    "fx_det_parts_f32_workspace": (_sz, [_i64, _i32]),
    "fx_det_parts_f32": (ctypes.c_int, [_p, _i64, _i32, _p, _p, _p, _i32, _p, _sz, _p]),
    "fx_slogpf_f32_workspace": (_sz, [_i64, _i32]),
    "fx_slogpf_f32": (ctypes.c_int, [_p, _i64, _i32, _i32, _p, _p, _p, _sz, _p]),
    "fx_pf_block_columns": (_i32, [_i32]),
    "fx_slogpf_factors_f32_workspace": (_sz, [_i64, _i32]),
    "fx_slogpf_factors_f32": (ctypes.c_int, [_p, _i64, _i32, _i32, _p, _p, _p, _p, _p, _p, _sz, _p]),
    "fx_slogpf_inverse_f32_workspace": (_sz, [_i64, _i32]),
    "fx_slogpf_inverse_f32": (ctypes.c_int, [_p, _p, _p, _p, _i64, _i32, _i32, _p, _i32, _p, _sz, _p]),
    "fx_slogpf_parts_f32_workspace": (_sz, [_i64, _i32]),
    "fx_slogpf_parts_f32": (ctypes.c_int, [_p, _i64, _i32, _i32, _i32, _p, _p, _p, _i32, _p, _sz, _p]),
    "fx_slogdet_f64_workspace": (_sz, [_i64, _i32]),
    "fx_slogdet_f64": (ctypes.c_int, [_p, _i64, _i32, _p, _p, _p, _sz, _p]),
    "fx_slogdet_parts_f64_workspace": (_sz, [_i64, _i32]),
    "fx_slogdet_parts_f64": (ctypes.c_int, [_p, _i64, _i32, _p, _p, _p, _p, _sz, _p]),
    "fx_slogpf_f64_workspace": (_sz, [_i64, _i32]),
    "fx_slogpf_f64": (ctypes.c_int, [_p, _i64, _i32, _i32, _p, _p, _p, _sz, _p]),
    "fx_slogpf_parts_f64_workspace": (_sz, [_i64, _i32]),
    "fx_slogpf_parts_f64": (ctypes.c_int, [_p, _i64, _i32, _i32, _i32, _p, _p, _p, _p, _sz, _p]),
}
# complex64 / complex128: the float64 signatures with interleaved (re, im) buffers;
# complex64's take the prec word before the workspace (PREC_ARG[_k]: the extra argument)
PREC_ARG = {"c64": [_i32], "c128": []}
for _k in ("c64", "c128"):
    _q = PREC_ARG[_k]
    SIGNATURES.update({
        f"fx_slogdet_{_k}_workspace": (_sz, [_i64, _i32]),
        f"fx_slogdet_{_k}": (ctypes.c_int, [_p, _i64, _i32, _p, _p] + _q + [_p, _sz, _p]),
        f"fx_slogdet_parts_{_k}_workspace": (_sz, [_i64, _i32]),
        f"fx_slogdet_parts_{_k}": (ctypes.c_int, [_p, _i64, _i32, _p, _p, _p] + _q + [_p, _sz, _p]),
        f"fx_slogpf_{_k}_workspace": (_sz, [_i64, _i32]),
        f"fx_slogpf_{_k}": (ctypes.c_int, [_p, _i64, _i32, _i32, _p, _p] + _q + [_p, _sz, _p]),
        f"fx_slogpf_parts_{_k}_workspace": (_sz, [_i64, _i32]),
        f"fx_slogpf_parts_{_k}": (ctypes.c_int, [_p, _i64, _i32, _i32, _i32, _p, _p, _p] + _q + [_p, _sz, _p]),
    })
# det's gradient (the exact adjugate) for the 64-bit and complex kinds
for _k in ("f64", "c64", "c128"):
    SIGNATURES.update({
        f"fx_det_parts_{_k}_workspace": (_sz, [_i64, _i32]),
        f"fx_det_parts_{_k}": (ctypes.c_int, [_p, _i64, _i32, _p, _p, _p] + PREC_ARG.get(_k, []) + [_p, _sz, _p]),
    })


# ------------------------------------------------- the network in front (include/fermix.h)

# element types
FX_F32, FX_F64, FX_BF16, FX_F16 = 0, 1, 2, 3
FX_MAX_RADIUS = 2048
FX_MAX_BIAS_HEADS = 4096
FX_MAX_POSITIONS = 1 << 30
FX_MAX_STEP_TOKENS = 0x7FFFFF00
FX_MIN_SCALE, FX_MAX_SCALE = 1e-30, 1e30
FX_NORM_LAYER, FX_NORM_POST, FX_NORM_PRE = 1, 2, 4
FX_MAX_COLUMNS = 8192


def _struct(name, layout):
    """A ctypes structure from lines of "type: fields"."""
    kinds = {"p": _p, "i64": _i64, "i32": _i32, "f32": ctypes.c_float}
    fields = [(f, kinds[k]) for line in layout.strip().splitlines() for k, fs in [line.split(":")] for f in fs.split()]
    return type(name, (ctypes.Structure,), {"_fields_": fields})


FxAttention = _struct("FxAttention", """
i64: batch
i32: nq nk heads kv_heads dim dtype causal offset radius buckets
f32: scale
p: q k v
i64: qb qn qh kb kn kh vb vn vh
p: table map q_pos k_pos lengths q_lengths mask out out_low stats grad_out grad_q grad_k grad_v grad_table
""")

FxAttentionStep = _struct("FxAttentionStep", """
i64: batch
i32: heads kv_heads dim dtype
i64: pages
i32: page_size max_pages radius buckets
f32: scale
p: q k v k_cache v_cache page_table lengths table map out
""")

FxResidualNorm = _struct("FxResidualNorm", """
i64: samples rows
i32: columns dtype wdtype flags
f32: eps alpha
p: x h gate
i64: xs xr hs hr gs gr gc os or_
p: post_weight post_bias scale pre_weight pre_bias y z stats
p: grad_y grad_z grad_x grad_h grad_gate
p: grad_post_weight grad_post_bias grad_scale grad_pre_weight grad_pre_bias
""")

for _n, _s in (("attention", FxAttention), ("residual_norm", FxResidualNorm)):
    _sp = ctypes.POINTER(_s)
    SIGNATURES[f"fx_{_n}_forward"] = (ctypes.c_int, [_sp, _p])
    SIGNATURES[f"fx_{_n}_grad_workspace"] = (_sz, [_sp])
    SIGNATURES[f"fx_{_n}_grad"] = (ctypes.c_int, [_sp, _p, _sz, _p])
SIGNATURES["fx_attention_keeps_low"] = (_i32, [ctypes.POINTER(FxAttention)])
SIGNATURES.update({
    "fx_relative_bias": (ctypes.c_int, [_p, _p, _i32, _i32, _p, _p, _i64, _i32, _i32, _i32, _i32, _p, _p]),
    "fx_relative_bias_grad_workspace": (_sz, [_i32, _i64, _i32, _i32, _i32, _i32]),
    "fx_relative_bias_grad": (
        ctypes.c_int,
        [_p, _p, _i32, _i32, _p, _p, _i64, _i32, _i32, _i32, _i32, _p, _p, _sz, _p],
    ),
    "fx_attention_step_workspace": (_sz, [ctypes.POINTER(FxAttentionStep)]),
    "fx_attention_step_run": (ctypes.c_int, [ctypes.POINTER(FxAttentionStep), _p, _sz, _p]),
})


class FermixLibraryError(RuntimeError):
    """The HIP library is missing, fails to load, or a call returned an error status."""


_lib = None


def lib():
    """The loaded library (loaded once). Raises FermixLibraryError if it is missing."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FermixLibraryError(
                f"{LIB_PATH} is missing: build it with `python -m fermix_amd.build` "
                "(fermix_amd has no non-HIP fallback)"
            )
        try:
            h = ctypes.CDLL(LIB_PATH)
        except OSError as e:  # pragma: no cover - environment specific
            raise FermixLibraryError(f"cannot load {LIB_PATH}: {e}") from e
        for name, (res, args) in SIGNATURES.items():
            f = getattr(h, name)
            f.restype = res
            f.argtypes = args
        _lib = h
    return _lib


def check(status, what):
    if status != FX_OK:
        msg = lib().fx_status_string(status).decode()
        raise FermixLibraryError(f"{what}: {msg} (status {status})")
