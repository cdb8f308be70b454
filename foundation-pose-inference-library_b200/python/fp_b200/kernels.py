"""ctypes bindings for the fpk_* kernel-level C ABI (include/fpk.h).

Device buffers are passed as integer addresses (e.g. ``tensor.data_ptr()``);
streams as integer ``cudaStream_t`` handles (0 = legacy default stream).
Every wrapper raises :class:`FpkError` with the library's message on failure.
"""
from __future__ import annotations

import ctypes as C
import math
import os
from pathlib import Path

PKG = Path(__file__).resolve().parents[2]
LIB_PATH = PKG / "lib" / "libfoundation_pose_nvidia.so"

FPK_DTYPE_F32 = 0
FPK_DTYPE_F16 = 1
FPK_DTYPE_BF16 = 2
FPK_DTYPE_F32_EXACT = 3  # fp32 kept exact (strict-FP32 networks)
FPK_DTYPE_E4M3 = 4  # element type of a KvCache only
FPK_ERROR_SLOT = 41  # codes that the calls with device-side indexes leave in their error flag
FPK_ERROR_PAGE = 42
FPK_ERROR_STARTS = 43
FPK_ERROR_LENGTH = 44
FPK_STATS_INTS = 8 + 65536


class FpkError(RuntimeError):
    pass


class Params(C.Structure):
    _fields_ = [
        ("depth_min", C.c_float), ("depth_max", C.c_float),
        ("erosion_radius", C.c_int), ("bilateral_radius", C.c_int),
        ("depth_diff_threshold", C.c_float), ("erosion_ratio_threshold", C.c_float),
        ("bilateral_sigma_d", C.c_float), ("bilateral_sigma_r", C.c_float),
        ("crop_ratio", C.c_float),
        ("input_width", C.c_int), ("input_height", C.c_int),
        ("rotation_normalizer_rad", C.c_float), ("znear", C.c_float), ("zfar", C.c_float),
        ("ambient_weight", C.c_float), ("diffuse_weight", C.c_float),
    ]


class Intrinsics(C.Structure):
    _fields_ = [("fx", C.c_float), ("fy", C.c_float), ("cx", C.c_float), ("cy", C.c_float)]


class Mesh(C.Structure):
    _fields_ = [
        ("vertices", C.c_void_p), ("normals", C.c_void_p), ("colors", C.c_void_p),
        ("uvs", C.c_void_p), ("texture", C.c_void_p), ("faces", C.c_void_p),
        ("n_vertices", C.c_int), ("n_faces", C.c_int),
        ("texture_width", C.c_int), ("texture_height", C.c_int),
    ]


_P = C.c_void_p
_SIGS = {
    "fpk_last_error": (C.c_char_p, []),
    "fpk_default_params": (None, [C.POINTER(Params)]),
    "fpk_preprocess": (C.c_int, [_P, _P, C.c_int, C.c_int, Intrinsics, C.POINTER(Params),
                                 _P, _P, _P, _P, _P]),
    "fpk_seed_poses": (C.c_int, [_P, _P, C.c_int, Intrinsics, C.POINTER(Params), _P, _P, _P]),
    "fpk_crop_boxes": (C.c_int, [_P, C.c_int, Intrinsics, C.c_float, C.POINTER(Params), _P, _P]),
    "fpk_render_workspace_bytes": (C.c_size_t, [C.c_int, C.c_int, C.POINTER(Params)]),
    "fpk_render": (C.c_int, [C.POINTER(Mesh), _P, _P, C.c_int, Intrinsics, C.POINTER(Params),
                             _P, _P, _P, _P, C.c_size_t, _P]),
    "fpk_pack": (C.c_int, [_P, _P, C.c_int, C.c_int, Intrinsics, C.POINTER(Params), _P, _P, _P,
                           _P, C.c_int, C.c_float, C.c_float, _P, _P, _P]),
    "fpk_render_pack": (C.c_int, [C.POINTER(Mesh), _P, C.c_int, _P, _P, C.c_int, C.c_int,
                                  Intrinsics, C.POINTER(Params), C.c_float, C.c_float, C.c_int,
                                  _P, C.c_longlong, _P, _P, C.c_size_t, _P]),
    "fpk_apply_deltas": (C.c_int, [_P, _P, _P, C.c_int, C.c_float, C.POINTER(Params), _P]),
    "fpk_select_best": (C.c_int, [_P, _P, C.c_int, C.POINTER(C.c_float), _P, _P]),
    "fpk_gemm": (C.c_int, [_P, _P]),
    "fpk_gemm_set_cta_pairs": (C.c_int, [C.c_int]),
    "fpk_gemm_set_tma_store": (C.c_int, [C.c_int]),
    "fpk_gemm_test_withhold_loads": (C.c_int, [C.c_int]),
    "fpk_attention": (C.c_int, [_P, C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_int, _P, C.c_longlong,
                                C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, _P, _P]),
    "fpk_qk_norm_rotary": (C.c_int, [_P, _P]),
    "fpk_cache_write": (C.c_int, [_P, _P]),
    "fpk_cache_read": (C.c_int, [_P, _P]),
    "fpk_attention_packed_workspace_bytes": (C.c_longlong, [_P]),
    "fpk_attention_packed": (C.c_int, [_P, _P]),
    "fpk_attention_paged_workspace_bytes": (C.c_longlong, [_P]),
    "fpk_attention_paged": (C.c_int, [_P, _P]),
    "fpk_attention_test_fail_share": (C.c_int, [C.c_int]),
    "fpk_net_create": (C.c_void_p, [C.c_char_p, C.c_char_p, C.c_int, C.c_int]),
    "fpk_net_destroy": (None, [_P]),
    "fpk_net_refine": (C.c_int, [_P, _P, _P, C.c_int, _P, _P, _P]),
    "fpk_net_score": (C.c_int, [_P, _P, _P, C.c_int, _P, _P]),
    "fpk_net_error": (C.c_int, [_P, C.POINTER(C.c_int)]),
}


def exported_symbols() -> list[str]:
    return list(_SIGS)


class FpkLibrary:
    def __init__(self, path: str | os.PathLike | None = None):
        self.path = Path(path) if path else LIB_PATH
        if not self.path.is_file():
            raise FpkError(f"{self.path} is not built (run foundation-pose-inference-library_b200/build.py)")
        self.lib = C.CDLL(str(self.path))
        for name, (res, args) in _SIGS.items():
            fn = getattr(self.lib, name)
            fn.restype = res
            fn.argtypes = args

    def _check(self, rc: int, what: str) -> None:
        if rc != 0:
            raise FpkError(f"{what}: {self.lib.fpk_last_error().decode()}")

    def default_params(self) -> Params:
        p = Params()
        self.lib.fpk_default_params(C.byref(p))
        return p

    def preprocess(self, depth_raw, mask, width, height, k, params, depth_filtered, eroded=0,
                   xyz=0, stats=0, stream=0):
        self._check(self.lib.fpk_preprocess(depth_raw, mask or None, width, height, k,
                                            C.byref(params), depth_filtered, eroded or None,
                                            xyz or None, stats or None, stream or None),
                    "fpk_preprocess")

    def seed_poses(self, stats, rotations, n, k, params, t0, poses, stream=0):
        self._check(self.lib.fpk_seed_poses(stats, rotations, n, k, C.byref(params), t0 or None,
                                            poses, stream or None), "fpk_seed_poses")

    def crop_boxes(self, poses, n, k, diameter, params, boxes, stream=0):
        self._check(self.lib.fpk_crop_boxes(poses, n, k, diameter, C.byref(params), boxes,
                                            stream or None), "fpk_crop_boxes")

    def render_workspace_bytes(self, n, n_vertices, params) -> int:
        return int(self.lib.fpk_render_workspace_bytes(n, n_vertices, C.byref(params)))

    def render(self, mesh, poses, boxes, n, k, params, out_rgb, out_xyz, tri_ids=0, stream=0,
               workspace=0, workspace_bytes=0):
        """workspace 0: the library allocates it stream-ordered for the call."""
        self._check(self.lib.fpk_render(C.byref(mesh), poses, boxes, n, k, C.byref(params),
                                        out_rgb, out_xyz, tri_ids or None, workspace or None,
                                        workspace_bytes, stream or None),
                    "fpk_render")

    def pack(self, rgb, depth_filtered, width, height, k, params, rend_rgb, rend_xyz, poses,
             boxes, n, diameter, invalid_threshold, net_r, net_o, stream=0):
        self._check(self.lib.fpk_pack(rgb, depth_filtered, width, height, k, C.byref(params),
                                      rend_rgb, rend_xyz, poses, boxes, n, diameter,
                                      invalid_threshold, net_r, net_o, stream or None),
                    "fpk_pack")

    def render_pack(self, mesh, poses, n, rgb, depth_filtered, width, height, k, params,
                    diameter, invalid_threshold, dtype, net, plane_stride, boxes, stream=0,
                    workspace=0, workspace_bytes=0):
        self._check(self.lib.fpk_render_pack(C.byref(mesh), poses, n, rgb, depth_filtered, width,
                                             height, k, C.byref(params), diameter,
                                             invalid_threshold, dtype, net, plane_stride,
                                             boxes or None, workspace or None, workspace_bytes,
                                             stream or None), "fpk_render_pack")

    def apply_deltas(self, poses, dt, dr, n, diameter, params, stream=0):
        self._check(self.lib.fpk_apply_deltas(poses, dt, dr, n, diameter, C.byref(params),
                                              stream or None), "fpk_apply_deltas")

    def select_best(self, poses, scores, n, center3, result, stream=0):
        c = (C.c_float * 3)(*[float(v) for v in center3])
        self._check(self.lib.fpk_select_best(poses, scores, n, c, result, stream or None),
                    "fpk_select_best")


FPK_DST_SAME = 0
FPK_DST_S2D = 1
FPK_DST_CONCAT = 2
FPK_DST_TOKENS = 3


class GemmDesc(C.Structure):
    _fields_ = [
        ("a", C.c_void_p), ("a_plane_stride", C.c_longlong), ("rows", C.c_int), ("cin", C.c_int),
        ("taps", C.c_int), ("tap_off", C.c_int * 16), ("w", C.c_void_p), ("cout", C.c_int),
        ("bias", C.c_void_p), ("residual", C.c_void_p), ("res_plane_stride", C.c_longlong),
        ("relu", C.c_int), ("dst", C.c_void_p), ("dst_plane_stride", C.c_longlong),
        ("dst_mode", C.c_int), ("img_rows", C.c_int), ("grid_w", C.c_int), ("valid_h", C.c_int),
        ("valid_w", C.c_int), ("dst_img_rows", C.c_int), ("dst_grid_w", C.c_int),
        ("img_mod", C.c_int), ("ch_step", C.c_int), ("pos", C.c_void_p), ("dtype", C.c_int),
        ("error_flag", C.c_void_p), ("splitk_ws", C.c_void_p), ("splitk_ws_bytes", C.c_longlong),
    ]


def _bind_gemm(lib) -> None:
    lib.fpk_gemm.restype = C.c_int
    lib.fpk_gemm.argtypes = [C.POINTER(GemmDesc), C.c_void_p]


def gemm(fl: "FpkLibrary", desc: GemmDesc, stream=0) -> None:
    if not getattr(fl, "_gemm_bound", False):
        _bind_gemm(fl.lib)
        fl._gemm_bound = True
    fl._check(fl.lib.fpk_gemm(C.byref(desc), stream or None), "fpk_gemm")


def attention(fl: FpkLibrary, qkv: int, qkv_plane_stride: int, qkv_layer_channels: int, q_channel: int,
              k_channel: int, v_channel: int, out: int, out_plane_stride: int, out_layer_channels: int,
              layers: int, heads: int, seq_len: int, n_seq: int, dtype: int, error_flag: int,
              stream: int | None = None) -> None:
    """fpk_attention: multi-head self-attention over planar activations (see include/fpk.h)."""
    fl._check(fl.lib.fpk_attention(qkv, qkv_plane_stride, qkv_layer_channels, q_channel, k_channel, v_channel,
                                   out, out_plane_stride, out_layer_channels, layers, heads, seq_len, n_seq,
                                   dtype, error_flag, stream or None), "fpk_attention")


class Heads(C.Structure):
    """fpk_heads_t: rows of heads, strides in bytes. Heads.planar and Heads.rows fill it in."""
    _fields_ = [("data", C.c_void_p), ("head_stride", C.c_longlong), ("row_stride", C.c_longlong),
                ("plane_stride", C.c_longlong)]

    @classmethod
    def planar(cls, data: int, plane_stride: int, head_dim: int, channel: int = 0) -> "Heads":
        """Heads from `channel` on of 16-bit planar activations (row 0 of plane 0 at `data`)."""
        return cls(data + channel // 8 * plane_stride, head_dim // 8 * plane_stride, 16, plane_stride)

    @classmethod
    def rows(cls, data: int, row_channels: int, head_dim: int, channel: int = 0) -> "Heads":
        """Heads from `channel` on of 16-bit rows of `row_channels` channels."""
        return cls(data + channel * 2, head_dim * 2, row_channels * 2, 16)


class QkRotaryDesc(C.Structure):
    _fields_ = [
        ("q", Heads), ("k", Heads), ("q_out", Heads), ("k_out", Heads), ("rows", C.c_int), ("q_heads", C.c_int),
        ("kv_heads", C.c_int), ("head_dim", C.c_int), ("rotary_dim", C.c_int), ("interleaved", C.c_int),
        ("q_weight", C.c_void_p), ("k_weight", C.c_void_p), ("eps", C.c_float), ("positions", C.c_void_p),
        ("inv_freq", C.c_void_p), ("rotary_scale", C.c_float), ("dtype", C.c_int),
    ]


class KvCache(C.Structure):
    _fields_ = [
        ("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("n_pages", C.c_int),
        ("page_rows", C.c_int), ("kv_heads", C.c_int), ("head_dim", C.c_int), ("dtype", C.c_int),
    ]


class CacheCopyDesc(C.Structure):
    _fields_ = [("cache", KvCache), ("k", Heads), ("v", Heads), ("rows", C.c_int), ("slots", C.c_void_p),
                ("dtype", C.c_int), ("error_flag", C.c_void_p)]


class PackedAttentionDesc(C.Structure):
    _fields_ = [
        ("q", Heads), ("k", Heads), ("v", Heads), ("out", Heads), ("q_heads", C.c_int), ("kv_heads", C.c_int),
        ("head_dim", C.c_int), ("n_seq", C.c_int), ("q_rows", C.c_int), ("kv_rows", C.c_int), ("q_starts", C.c_void_p),
        ("kv_starts", C.c_void_p), ("causal", C.c_int), ("scale", C.c_float), ("dtype", C.c_int),
        ("error_flag", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_longlong),
    ]


class PagedAttentionDesc(C.Structure):
    _fields_ = [
        ("q", Heads), ("out", Heads), ("cache", KvCache), ("q_heads", C.c_int), ("n_seq", C.c_int), ("q_rows", C.c_int),
        ("q_starts", C.c_void_p), ("kv_lengths", C.c_void_p), ("page_table", C.c_void_p), ("table_pages", C.c_int),
        ("causal", C.c_int), ("scale", C.c_float), ("dtype", C.c_int), ("error_flag", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_longlong),
    ]


def qk_norm_rotary(fl: FpkLibrary, desc: QkRotaryDesc, stream=0) -> None:
    """fpk_qk_norm_rotary: RMS norm of query and key heads and rotary positions (include/fpk.h)."""
    fl._check(fl.lib.fpk_qk_norm_rotary(C.byref(desc), stream or None), "fpk_qk_norm_rotary")


def cache_write(fl: FpkLibrary, desc: CacheCopyDesc, stream=0) -> None:
    """fpk_cache_write: rows of keys and values into slots of a paged cache."""
    fl._check(fl.lib.fpk_cache_write(C.byref(desc), stream or None), "fpk_cache_write")


def cache_read(fl: FpkLibrary, desc: CacheCopyDesc, stream=0) -> None:
    """fpk_cache_read: slots of a paged cache back into rows of keys and values."""
    fl._check(fl.lib.fpk_cache_read(C.byref(desc), stream or None), "fpk_cache_read")


def attention_packed_workspace_bytes(fl: FpkLibrary, desc: PackedAttentionDesc) -> int:
    return int(fl.lib.fpk_attention_packed_workspace_bytes(C.byref(desc)))


def attention_packed(fl: FpkLibrary, desc: PackedAttentionDesc, stream=0) -> None:
    """fpk_attention_packed: attention within packed sequences of different lengths."""
    fl._check(fl.lib.fpk_attention_packed(C.byref(desc), stream or None), "fpk_attention_packed")


def attention_paged_workspace_bytes(fl: FpkLibrary, desc: PagedAttentionDesc) -> int:
    return int(fl.lib.fpk_attention_paged_workspace_bytes(C.byref(desc)))


def attention_paged(fl: FpkLibrary, desc: PagedAttentionDesc, stream=0) -> None:
    """fpk_attention_paged: attention of each sequence's newest rows over its cached keys and values."""
    fl._check(fl.lib.fpk_attention_paged(C.byref(desc), stream or None), "fpk_attention_paged")


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, factor: float = 1.0, trained_length: int = 0,
                       slow_turns: float = 1.0, fast_turns: float = 32.0) -> list[float]:
    """The table inv_freq of fpk_qk_norm_rotary: base^(-2i/rotary_dim), i < rotary_dim/2.

    For contexts `factor` times as long as the trained ones: with trained_length 0 every frequency
    is divided by factor (positions are interpolated). With trained_length given, only slow
    frequencies are: those that turn fewer than slow_turns times over the trained length are divided
    whole, those above fast_turns are kept, and between the two the share kept grows linearly.
    """
    if rotary_dim <= 0 or rotary_dim % 2 or base <= 0 or factor <= 0 or fast_turns <= slow_turns:
        raise ValueError("rotary_frequencies: rotary_dim must be even, base and factor positive, fast_turns above slow_turns")
    out = []
    for i in range(rotary_dim // 2):
        f = base ** (-2.0 * i / rotary_dim)
        kept = 0.0
        if trained_length > 0:
            turns = trained_length * f / (2.0 * math.pi)
            kept = min(1.0, max(0.0, (turns - slow_turns) / (fast_turns - slow_turns)))
        out.append(f * kept + f / factor * (1.0 - kept))
    return out


class Networks:
    """RefineNet + ScoreNet handle (fpk_net_*); precision 2 = FP16, 3 = BF16."""

    def __init__(self, fl: FpkLibrary, refine_pack, score_pack, precision: int, max_batch: int):
        self.fl = fl
        self.h = fl.lib.fpk_net_create(str(refine_pack).encode(), str(score_pack).encode(),
                                       int(precision), int(max_batch))
        if not self.h:
            raise FpkError(f"fpk_net_create: {fl.lib.fpk_last_error().decode()}")

    def refine(self, rendered, observed, n, trans, rot, stream=0):
        self.fl._check(self.fl.lib.fpk_net_refine(self.h, rendered, observed, n, trans, rot,
                                                  stream or None), "fpk_net_refine")

    def score(self, rendered, observed, n, scores, stream=0):
        self.fl._check(self.fl.lib.fpk_net_score(self.h, rendered, observed, n, scores,
                                                 stream or None), "fpk_net_score")

    def error_flag(self) -> int:
        v = C.c_int(0)
        self.fl._check(self.fl.lib.fpk_net_error(self.h, C.byref(v)), "fpk_net_error")
        return v.value

    def close(self):
        if self.h:
            self.fl.lib.fpk_net_destroy(self.h)
            self.h = None

    __del__ = close
