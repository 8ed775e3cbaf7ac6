"""Python host side of the trmoe C ABI (include/trmoe.h) — ctypes bindings plus a small layer
object that keeps one MoE layer's weights in HBM.

This mirrors the reference's Rust call sites (tr_model::exec::Model::moe_block /
exec_batch::moe_batch) for tests and the benchmark; device memory and streams come from torch.
There is no CPU fallback: without the built HIP library every entry point raises.
"""
from __future__ import annotations

import ctypes as C
import functools
import os

HERE = os.path.dirname(os.path.abspath(__file__))
PKG_ROOT = os.path.dirname(HERE)
LIB_PATH = os.path.join(PKG_ROOT, "libtrmoe.so")
HEADER = os.path.join(os.path.dirname(PKG_ROOT), "include", "trmoe.h")

FMT_Q4_K, FMT_Q6_K, FMT_Q8_0, FMT_Q5_1 = 12, 14, 8, 7
# the reference's TQ codecs (codec.rs:1-46): bits << 8 | kb
FMT_TQ4_16, FMT_TQ4_32, FMT_TQ5_16, FMT_TQ5_32, FMT_TQ8_16, FMT_TQ8_32 = 0x410, 0x420, 0x510, 0x520, 0x810, 0x820
TQ_FMTS = (FMT_TQ4_16, FMT_TQ4_32, FMT_TQ5_16, FMT_TQ5_32, FMT_TQ8_16, FMT_TQ8_32)
BASIS_ALL, BASIS_TOP = 0, 1
DT_F32, DT_BF16, DT_F16 = 0, 1, 2
SCORES = {"softmax": 0, "sigmoid": 1}
K_MAX = 32
(WS_RLOG, WS_IDS, WS_W, WS_NSEL, WS_ENT_TOK, WS_ENT_W, WS_ENT_EXP, WS_GRP_START, WS_GRP_EXP, WS_NGROUPS, WS_XQ,
 WS_XS, WS_ACTQ, WS_ACTS, WS_SHLOGIT, WS_BARRIER_ERR, WS_MIXED) = range(1, 18)


class TrkError(RuntimeError):
    pass


class Mat(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("rows", C.c_uint32), ("k", C.c_uint32), ("fmt", C.c_uint32),
                ("count", C.c_uint32), ("stride", C.c_uint64), ("tile_stride", C.c_uint64)]


class HcW(C.Structure):
    """trk_hc_w: the hyper-connection up projection [hc * hidden][lr] (a kb-32 TQ codec)."""
    _fields_ = [("up", Mat), ("hc", C.c_uint32), ("lr", C.c_uint32)]


class MoeW(C.Structure):
    _fields_ = [("router", C.c_void_p), ("router_bias", C.c_void_p), ("shexp_gate", C.c_void_p),
                ("gate", Mat), ("up", Mat), ("down", Mat), ("sh_gate", Mat), ("sh_up", Mat), ("sh_down", Mat)]


class Policy(C.Structure):
    _fields_ = [("min", C.c_uint32), ("max", C.c_uint32), ("mass", C.c_float), ("basis", C.c_uint32)]


class ScorePolicy(C.Structure):
    """trk_score_policy: how trk_route_scores chooses."""
    _fields_ = [("k", C.c_uint32), ("score", C.c_uint32), ("n_group", C.c_uint32), ("topk_group", C.c_uint32),
                ("group_top", C.c_uint32), ("renorm", C.c_int32), ("factor", C.c_float)]


class I8Mat(C.Structure):
    """trk_i8_mat: a stack of int8 matrices with a scale per row."""
    _fields_ = [("ptr", C.c_void_p), ("scale", C.c_void_p), ("rows", C.c_uint32), ("k", C.c_uint32),
                ("count", C.c_uint32), ("ld", C.c_uint64), ("stride", C.c_uint64)]


class Mx4Mat(C.Structure):
    """trk_mx4_mat: a stack of 4-bit matrices with a power of two for each 32 values of a row."""
    _fields_ = [("ptr", C.c_void_p), ("scale", C.c_void_p), ("rows", C.c_uint32), ("k", C.c_uint32),
                ("count", C.c_uint32), ("ld", C.c_uint64), ("stride", C.c_uint64), ("scale_ld", C.c_uint64),
                ("scale_stride", C.c_uint64)]


class MoeMx4W(C.Structure):
    """trk_moe_mx4_w: a MoE layer on 4-bit experts."""
    _fields_ = [("router", C.c_void_p), ("bias", C.c_void_p), ("shared_gate", C.c_void_p), ("gate", Mx4Mat),
                ("up", Mx4Mat), ("down", Mx4Mat), ("n_shared", C.c_uint32)]


class Cfg(C.Structure):
    _fields_ = [("hidden", C.c_uint32), ("n_expert", C.c_uint32), ("n_ff", C.c_uint32),
                ("n_expert_used", C.c_uint32), ("m_max", C.c_uint32), ("k_cap", C.c_uint32),
                ("router_dot_max_m", C.c_uint32), ("hiprec", C.c_int32), ("n_tiles", C.c_uint32),
                ("n_expert_packed", C.c_uint32)]


class Stats(C.Structure):
    _fields_ = [("rows", C.c_uint64), ("experts", C.c_uint64)]


_lib = None


def lib() -> C.CDLL:
    """Load libtrmoe.so (built by `make -C tr-infer_amd` / __graft_entry__.build())."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise TrkError(f"{LIB_PATH} is not built: run __graft_entry__.build() (make -C tr-infer_amd)")
        L = C.CDLL(LIB_PATH)
        vp, u32, u64, i, f, sz = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int, C.c_float, C.c_size_t
        L.trk_last_error.restype = C.c_char_p
        L.trk_create.argtypes = [C.POINTER(Cfg), C.POINTER(vp)]
        L.trk_workspace_bytes.argtypes = [C.POINTER(Cfg), u32, C.POINTER(sz)]
        L.trk_destroy.argtypes = [vp]
        L.trk_set_moe.argtypes = [vp, C.POINTER(Policy)]
        L.trk_moe_forward.argtypes = [vp, C.POINTER(MoeW), vp, vp, u32, vp, vp]
        L.trk_moe_residual.argtypes = [vp, C.POINTER(MoeW), vp, f, vp, u32, vp]
        L.trk_moe_forward_hc.argtypes = [vp, C.POINTER(MoeW), C.POINTER(HcW), vp, vp, u32, vp, vp]
        L.trk_moe_forward_noalloc.argtypes = [C.POINTER(Cfg), C.POINTER(Policy), C.POINTER(MoeW), vp, vp, u32, vp,
                                              vp]
        L.trk_get_stats.argtypes = [vp, C.POINTER(Stats), i, vp]
        L.trk_profile_start.argtypes = [vp, i, vp]
        L.trk_profile_report.argtypes = [vp, C.POINTER(C.c_double), C.POINTER(C.c_uint64), vp]
        L.trk_router_logits.argtypes = [vp, vp, vp, vp, u32, u32, u32, i, vp, vp, vp]
        L.trk_route.argtypes = [vp, u32, u32, u32, C.POINTER(Policy), vp, vp, vp, vp]
        L.trk_quantize.argtypes = [vp, u32, u32, u32, i, vp, vp, vp, vp]
        L.trk_gemv.argtypes = [C.POINTER(Mat), u32, u32, u32, u32, vp, vp, vp, u32, i, vp, u32, vp, i, vp]
        L.trk_route_scores.argtypes = [vp, vp, u32, u32, C.POINTER(ScorePolicy), vp, vp, vp, vp]
        L.trk_quantize_rows.argtypes = [vp, u32, u64, u32, u32, vp, u64, vp, vp]
        L.trk_gemm_i8.argtypes = [C.POINTER(I8Mat), u32, vp, u64, vp, u32, vp, vp, u32, u64, i, vp]
        L.trk_experts_plan_words.argtypes = [u32, u32, u32, C.POINTER(u64)]
        L.trk_experts_plan.argtypes = [vp, vp, u32, u32, u32, vp, vp]
        L.trk_experts_up_i8.argtypes = [C.POINTER(I8Mat), C.POINTER(I8Mat), vp, u64, vp, u32, vp, vp, u32, vp, vp, u32,
                                        u64, vp]
        L.trk_experts_down_work_bytes.argtypes = [u32, u32, u32, u32, C.POINTER(u64)]
        L.trk_experts_down_i8.argtypes = [C.POINTER(I8Mat), vp, u64, vp, u32, vp, vp, vp, u32, vp, vp, vp, u32, u64, i,
                                          vp]
        L.trk_quantize_mx4.argtypes = [vp, u32, u64, u32, u32, vp, u64, vp, u64, vp]
        L.trk_dequantize_mx4.argtypes = [vp, u64, vp, u64, u32, u32, vp, u32, u64, vp]
        L.trk_gemm_mx4.argtypes = [C.POINTER(Mx4Mat), u32, vp, u64, vp, u64, u32, vp, vp, u32, u64, i, vp]
        L.trk_experts_up_mx4.argtypes = [C.POINTER(Mx4Mat), C.POINTER(Mx4Mat), vp, u64, vp, u64, u32, vp, vp, u32, vp, vp,
                                         u32, u64, vp]
        L.trk_experts_down_mx4.argtypes = [C.POINTER(Mx4Mat), vp, u64, vp, u64, u32, vp, vp, vp, u32, vp, vp, vp, u32, u64,
                                           i, vp]
        L.trk_moe_mx4_work_bytes.argtypes = [C.POINTER(MoeMx4W), u32, u32, C.POINTER(u64)]
        L.trk_moe_mx4.argtypes = [C.POINTER(MoeMx4W), C.POINTER(ScorePolicy), vp, u32, u64, vp, u32, vp, vp, u32, u64, vp]
        L.trk_swiglu.argtypes = [vp, vp, vp, sz, vp]
        L.trk_rmsnorm.argtypes = [vp, vp, f, u32, u32, vp, vp]
        L.trk_add_inplace.argtypes = [vp, vp, sz, vp]
        L.trk_gen_gguf.argtypes = [u32, u64, u64, u32, u32, f, f, vp, vp]
        L.trk_gen_gguf_stack.argtypes = [u32, u64, u64, u64, u32, u32, u32, f, f, vp, u64, vp]
        L.trk_gen_normal.argtypes = [u64, u64, sz, C.c_double, vp, vp]
        L.trk_debug_read.argtypes = [vp, i, vp, sz, vp]
        L.trk_launch_kernel.argtypes = [vp, C.POINTER(MoeW), vp, vp, u32, vp, C.c_char_p, vp]
        L.trk_set_timing.argtypes = [vp, i]
        L.trk_set_fusion.argtypes = [vp, i]
        L.trk_set_stream_rows.argtypes = [vp, i]
        L.trk_set_decode_rows.argtypes = [vp, i]
        L.trk_set_tq_mfma.argtypes = [vp, i]
        L.trk_get_timing.argtypes = [vp, C.POINTER(C.c_char_p), C.POINTER(C.c_double), C.POINTER(C.c_uint64), i]
        _lib = L
    return _lib


def check(rc: int) -> None:
    if rc != 0:
        raise TrkError(f"trmoe error {rc}: {lib().trk_last_error().decode()}")


def header_functions() -> list[str]:
    """Names of the functions include/trmoe.h declares."""
    import re
    txt = open(HEADER).read()
    return sorted(set(re.findall(r"^\s*(?:int|const char \*)\s*(trk_\w+)\s*\(", txt, re.M)))


def row_bytes(fmt: int, k: int) -> int:
    return k // 256 * {FMT_Q4_K: 144, FMT_Q6_K: 210, FMT_Q8_0: 272, FMT_Q5_1: 192}[fmt]


def tq_block_bytes(fmt: int) -> int:
    """Codec::block_bytes (codec.rs:22-29)."""
    bits, kb = fmt >> 8, fmt & 0xFF
    return 64 + (16 * kb if bits == 8 else 8 * kb) + (2 * kb if bits == 5 else 0)


def matrix_bytes(fmt: int, rows: int, k: int) -> int:
    """Bytes of one [rows][k] matrix: TQ strips (rows padded to 16) or GGUF rows."""
    if fmt in TQ_FMTS:
        return (rows + 15) // 16 * (k // (fmt & 0xFF)) * tq_block_bytes(fmt)
    return rows * row_bytes(fmt, k)


def _ptr(t):
    return None if t is None else t.data_ptr()


_current_raw_stream = None


def _stream(stream=None):
    """The hipStream_t of `stream`, or of torch's current stream on the current device.  The raw handle
    is asked for directly: a torch.cuda.Stream object for it costs 2.5 us, as much as a launch."""
    global _current_raw_stream
    if stream is not None:
        return stream.cuda_stream
    if _current_raw_stream is None:
        import torch
        torch.cuda.init()
        raw, dev = getattr(torch._C, "_cuda_getCurrentRawStream", None), getattr(torch._C, "_cuda_getDevice", None)
        if raw is not None and dev is not None:
            _current_raw_stream = lambda: raw(dev())  # noqa: E731
        else:
            _current_raw_stream = lambda: torch.cuda.current_stream().cuda_stream  # noqa: E731
    return _current_raw_stream()


class Context:
    """trk_create/trk_destroy around one layer shape (Model::load_with's workspace sizing)."""

    def __init__(self, hidden, n_expert, n_ff, k, m_max, k_cap=0, router_dot_max_m=16, hiprec=True, n_tiles=1,
                 n_expert_packed=0):
        self.cfg = Cfg(hidden, n_expert, n_ff, k, m_max, k_cap, router_dot_max_m, int(hiprec), n_tiles,
                       n_expert_packed)
        h = C.c_void_p()
        check(lib().trk_create(C.byref(self.cfg), C.byref(h)))
        self.h = h
        self.k = k

    def close(self):
        if self.h:
            lib().trk_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_moe(self, policy):
        """policy: None or (min, max, mass, basis) (Model::set_moe)."""
        if policy is None:
            check(lib().trk_set_moe(self.h, None))
        else:
            p = Policy(*policy)
            check(lib().trk_set_moe(self.h, C.byref(p)))

    def forward(self, w: "LayerWeights", x, out, rlog=None, stream=None):
        check(lib().trk_moe_forward(self.h, C.byref(w.moew), _ptr(x), _ptr(rlog), x.shape[0], _ptr(out),
                                    _stream(stream)))

    def forward_hc(self, w: "LayerWeights", up, hc, lr, xn, lo, out, stream=None):
        """trk_moe_forward_hc: out = MoE(the hyper-connection mix of xn [M][hc][H] and lo [M][lr]);
        up: a uint8 tensor holding the TQ matrix [hc * H][lr] in `up_fmt` = (bits << 8) | 32."""
        upt, fmt = up
        hw = HcW(Mat(upt.data_ptr(), hc * w.H, lr, fmt, 1, matrix_bytes(fmt, hc * w.H, lr)), hc, lr)
        check(lib().trk_moe_forward_hc(self.h, C.byref(w.moew), C.byref(hw), _ptr(xn), _ptr(lo), lo.shape[0],
                                       _ptr(out), _stream(stream)))

    def launch_kernel(self, name: str, w: "LayerWeights", x, out, rlog=None, stream=None):
        """Launch one kernel of the forward sequence (timing in isolation; see trk_launch_kernel)."""
        check(lib().trk_launch_kernel(self.h, C.byref(w.moew), _ptr(x), _ptr(rlog), x.shape[0], _ptr(out),
                                      name.encode(), _stream(stream)))

    def residual(self, w: "LayerWeights", rms_w, eps, h, stream=None):
        check(lib().trk_moe_residual(self.h, C.byref(w.moew), _ptr(rms_w), eps, _ptr(h), h.shape[0], _stream(stream)))

    def stats(self, reset=False, stream=None):
        """(rows, experts) routed since the last reset (MoeStats::snapshot); raises on TRK_E_TIMEOUT."""
        s = Stats()
        check(lib().trk_get_stats(self.h, C.byref(s), int(reset), _stream(stream)))
        return s.rows, s.experts

    def profile_start(self, on=True, stream=None):
        """MoeStats::profile_start: zero the router-mass profile and collect it on later forwards."""
        check(lib().trk_profile_start(self.h, int(on), _stream(stream)))

    def profile_report(self, stream=None):
        """MoeStats::profile_report: (mean cumulative mass of the best 1..32 experts, rows profiled)."""
        import numpy as np
        cum = np.zeros(K_MAX, np.float64)
        rows = C.c_uint64()
        check(lib().trk_profile_report(self.h, cum.ctypes.data_as(C.POINTER(C.c_double)), C.byref(rows),
                                       _stream(stream)))
        return cum, rows.value

    def set_fusion(self, on: bool):
        check(lib().trk_set_fusion(self.h, int(on)))

    def set_tq_mfma(self, on: bool):
        """TQ layers on the int8 MFMA kernels (True) or the generic grouped TQ GEMV (False)."""
        check(lib().trk_set_tq_mfma(self.h, int(bool(on))))

    def set_stream_rows(self, rows: int):
        """Batch items of at most `rows` rows on the streaming GEMV (-1 automatic, 0 none)."""
        check(lib().trk_set_stream_rows(self.h, int(rows)))

    def set_decode_rows(self, rows: int):
        """GGUF batches of 2..rows tokens as per-token decode units (0 never, default 8)."""
        check(lib().trk_set_decode_rows(self.h, int(rows)))

    def set_timing(self, on: bool):
        check(lib().trk_set_timing(self.h, int(on)))

    def timing(self):
        """{kernel: (total ms, launches)} since the last call (synchronises)."""
        cap = 16
        names = (C.c_char_p * cap)()
        ms = (C.c_double * cap)()
        cnt = (C.c_uint64 * cap)()
        n = lib().trk_get_timing(self.h, names, ms, cnt, cap)
        if n < 0:
            check(n)
        return {names[i].decode(): (ms[i], int(cnt[i])) for i in range(min(n, cap))}

    def read(self, which, nbytes, dtype, stream=None):
        import numpy as np
        buf = np.zeros(nbytes, np.uint8)
        check(lib().trk_debug_read(self.h, which, buf.ctypes.data_as(C.c_void_p), nbytes, _stream(stream)))
        return buf.view(dtype)


class LayerWeights:
    """One layer's weights resident on the GPU: expert stacks [E][rows*row_bytes] as uint8 tensors."""

    def __init__(self, H, E, F, router, shexp_gate, gate, up, down, sh_gate, sh_up, sh_down, gate_fmt=FMT_Q4_K,
                 down_fmt=FMT_Q4_K, router_bias=None):
        self.H, self.E, self.F = H, E, F
        self.tensors = dict(router=router, shexp_gate=shexp_gate, gate=gate, up=up, down=down, sh_gate=sh_gate,
                            sh_up=sh_up, sh_down=sh_down, router_bias=router_bias)
        gm, dmb = matrix_bytes(gate_fmt, F, H), matrix_bytes(down_fmt, H, F)

        def mat(t, rows, k, fmt, count, mb):
            return Mat(t.data_ptr(), rows, k, fmt, count, mb, 0)

        self.moew = MoeW(router.data_ptr() if router is not None else None,
                         router_bias.data_ptr() if router_bias is not None else None, shexp_gate.data_ptr(),
                         mat(gate, F, H, gate_fmt, E, gm), mat(up, F, H, gate_fmt, E, gm), mat(down, H, F, down_fmt, E, dmb),
                         mat(sh_gate, F, H, gate_fmt, 1, gm), mat(sh_up, F, H, gate_fmt, 1, gm),
                         mat(sh_down, H, F, down_fmt, 1, dmb))
        self.bytes_per_expert = 2 * gm + dmb

    @classmethod
    def from_host(cls, layer, device="cuda"):
        """Upload a host-side layer (raw GGUF bytes; see tests/layerdata.py)."""
        import numpy as np
        import torch

        def dev(a, dtype=None):
            return torch.from_numpy(np.ascontiguousarray(a)).to(device)

        return cls(layer.H, layer.E, layer.F, dev(layer.router), dev(layer.shexp_gate), dev(layer.stacked("gate")),
                   dev(layer.stacked("up")), dev(layer.stacked("down")), dev(layer.sh_gate), dev(layer.sh_up),
                   dev(layer.sh_down), layer.gate_fmt, layer.down_fmt,
                   None if layer.bias is None else dev(layer.bias))

    @classmethod
    def from_tq(cls, H, E, F, router, shexp_gate, gate, up, down, sh_gate, sh_up, sh_down, gate_fmt, down_fmt,
                router_bias=None, device="cuda"):
        """Upload a layer whose experts are the reference's packed TQ strips (host arrays: gate /
        up / down as [E][matrix bytes], the shared expert's as one matrix each), unchanged."""
        import numpy as np
        import torch

        def dev(a):
            return torch.from_numpy(np.ascontiguousarray(a)).to(device)

        return cls(H, E, F, dev(router), dev(shexp_gate), dev(gate), dev(up), dev(down), dev(sh_gate), dev(sh_up),
                   dev(sh_down), gate_fmt, down_fmt, None if router_bias is None else dev(router_bias))

    @classmethod
    def generate(cls, seed, layer, H, E, F, down_fmt=FMT_Q4_K, router_bias=None, device="cuda", stream=None):
        """Synthesise a layer on the GPU with the same generator the test oracle uses."""
        import torch
        gb, db = row_bytes(FMT_Q4_K, H), row_bytes(down_fmt, F)
        L = lib()
        st = _stream(stream)

        def sid(t):
            return (layer << 32) | t

        router = torch.empty(E * H, dtype=torch.float32, device=device)
        check(L.trk_gen_normal(seed, sid(1), E * H, 0.02, _ptr(router), st))
        shg = torch.empty(H, dtype=torch.float32, device=device)
        check(L.trk_gen_normal(seed, sid(2), H, 0.02, _ptr(shg), st))
        gate = torch.empty((E, F * gb), dtype=torch.uint8, device=device)
        up = torch.empty((E, F * gb), dtype=torch.uint8, device=device)
        down = torch.empty((E, H * db), dtype=torch.uint8, device=device)
        # expert e: gate / up / down from streams 16 + 3e, 17 + 3e, 18 + 3e of this layer
        for t, fmt, rows, k, buf in ((gate, FMT_Q4_K, F, H, 16), (up, FMT_Q4_K, F, H, 17), (down, down_fmt, H, F, 18)):
            check(L.trk_gen_gguf_stack(fmt, seed, sid(buf), 3, E, rows, k, 1e-4, 2e-3, _ptr(t), t.stride(0), st))
        sh_gate = torch.empty(F * gb, dtype=torch.uint8, device=device)
        sh_up = torch.empty(F * gb, dtype=torch.uint8, device=device)
        sh_down = torch.empty(H * db, dtype=torch.uint8, device=device)
        check(L.trk_gen_gguf(FMT_Q4_K, seed, sid(8), F, H, 1e-4, 2e-3, _ptr(sh_gate), st))
        check(L.trk_gen_gguf(FMT_Q4_K, seed, sid(9), F, H, 1e-4, 2e-3, _ptr(sh_up), st))
        check(L.trk_gen_gguf(down_fmt, seed, sid(10), H, F, 1e-4, 2e-3, _ptr(sh_down), st))
        return cls(H, E, F, router, shg, gate, up, down, sh_gate, sh_up, sh_down, FMT_Q4_K, down_fmt, router_bias)


    @classmethod
    def from_tiled_tq(cls, H, E, F, T, router, shexp_gate, gate, up, down, sh_gate, sh_up, sh_down, gate_fmt,
                      down_fmt, router_bias=None, device="cuda"):
        """A layer as a pack written for T tiles holds it (python/trpack/plan.py:106-118,174-181),
        uploaded unchanged: router [T][E][H/T]; gate / up [T][count][tile bytes] (tile t: rows
        [F/T t, F/T (t+1)) as a [F/T][H] TQ matrix), down [T][count][tile bytes] (columns
        [F/T t, F/T (t+1)), [H][F/T]); the shared expert's as [T][tile bytes].  count < E: a
        subset pack of the first `count` experts."""
        import numpy as np
        import torch

        def dev(a):
            return torch.from_numpy(np.ascontiguousarray(a)).to(device)

        self = cls.__new__(cls)
        self.H, self.E, self.F = H, E, F
        t = dict(router=dev(router), shexp_gate=dev(shexp_gate), gate=dev(gate), up=dev(up), down=dev(down),
                 sh_gate=dev(sh_gate), sh_up=dev(sh_up), sh_down=dev(sh_down),
                 router_bias=None if router_bias is None else dev(router_bias))
        self.tensors = t
        per = F // T

        def mat(name, rows, k, fmt):
            a = t[name]
            if a.dim() == 2:  # [T][bytes]: one matrix per tile
                return Mat(a.data_ptr(), rows, k, fmt, 1, a.shape[1], a.stride(0))
            return Mat(a.data_ptr(), rows, k, fmt, a.shape[1], a.stride(1), a.stride(0))

        self.moew = MoeW(t["router"].data_ptr(), None if router_bias is None else t["router_bias"].data_ptr(),
                         t["shexp_gate"].data_ptr(), mat("gate", per, H, gate_fmt), mat("up", per, H, gate_fmt),
                         mat("down", H, per, down_fmt), mat("sh_gate", per, H, gate_fmt),
                         mat("sh_up", per, H, gate_fmt), mat("sh_down", H, per, down_fmt))
        self.bytes_per_expert = T * (2 * matrix_bytes(gate_fmt, per, H) + matrix_bytes(down_fmt, H, per))
        return self

    @classmethod
    def generate_tq(cls, gen, H, E, F, gate_fmt=None, down_fmt=None, router_bias=None, device="cuda"):
        """A synthetic layer of packed TQ experts generated on the GPU from a torch Generator:
        router and shared-gate vector ~ N(0, 0.02), every TQ matrix as `gen_tq_stack`."""
        import torch
        gf = FMT_TQ4_32 if gate_fmt is None else gate_fmt
        df = FMT_TQ5_16 if down_fmt is None else down_fmt
        router = torch.randn((E, H), device=device, generator=gen) * 0.02
        shg = torch.randn(H, device=device, generator=gen) * 0.02
        gate, up = (gen_tq_stack(gen, E, F, H, gf, device) for _ in range(2))
        down = gen_tq_stack(gen, E, H, F, df, device)
        sg, su = (gen_tq_stack(gen, 1, F, H, gf, device)[0] for _ in range(2))
        sd = gen_tq_stack(gen, 1, H, F, df, device)[0]
        return cls(H, E, F, router, shg, gate, up, down, sg, su, sd, gf, df, router_bias)

    def with_down(self, down_fmt, seed, layer, device="cuda", stream=None):
        """The same layer with its routed and shared down projections regenerated in `down_fmt`
        (config 4: Q4_K gate/up, Q6_K down); every other tensor is shared with this one."""
        import torch
        H, E, F = self.H, self.E, self.F
        db = row_bytes(down_fmt, F)
        L = lib()
        st = _stream(stream)
        down = torch.empty((E, H * db), dtype=torch.uint8, device=device)
        check(L.trk_gen_gguf_stack(down_fmt, seed, (layer << 32) | 18, 3, E, H, F, 1e-4, 2e-3, _ptr(down),
                                   down.stride(0), st))
        sh_down = torch.empty(H * db, dtype=torch.uint8, device=device)
        check(L.trk_gen_gguf(down_fmt, seed, (layer << 32) | 10, H, F, 1e-4, 2e-3, _ptr(sh_down), st))
        t = self.tensors
        return LayerWeights(H, E, F, t["router"], t["shexp_gate"], t["gate"], t["up"], down, t["sh_gate"],
                            t["sh_up"], sh_down, FMT_Q4_K, down_fmt, t["router_bias"])


def gen_tq_stack(gen, count, rows, k, fmt, device="cuda"):
    """A stack of `count` packed TQ matrices [rows][k] on the GPU (codec.rs:1-46): uniform q bytes
    (and 5-bit planes), each block's f16 d in [5e-4, 3e-3] and m = -d * U(0, 2^(bits-1)), the sign
    pattern of converted GGUF weights.  `gen` is a torch Generator on `device`."""
    import torch
    mb = matrix_bytes(fmt, rows, k)
    bb, bits = tq_block_bytes(fmt), fmt >> 8
    t = torch.randint(0, 256, (count, mb), dtype=torch.uint8, device=device, generator=gen)
    blocks = t.view(count, mb // bb, bb)
    d = torch.empty((count, mb // bb, 16), device=device).uniform_(5e-4, 3e-3, generator=gen)
    m = -d * torch.empty_like(d).uniform_(0, float(1 << (bits - 1)), generator=gen)
    blocks[:, :, 0:32] = d.half().view(torch.uint8)
    blocks[:, :, 32:64] = m.half().view(torch.uint8)
    return t


NOALLOC_SCRATCH_BYTES = 16 << 20


def workspace_bytes(hidden, n_expert, n_ff, k, m, k_cap=0):
    """trk_workspace_bytes: the device workspace of the layer for m rows (host-side sizing)."""
    out = C.c_size_t()
    cfg = Cfg(hidden, n_expert, n_ff, k, m, k_cap, 16, 1)
    check(lib().trk_workspace_bytes(C.byref(cfg), m, C.byref(out)))
    return out.value


def noalloc_max_m(hidden, n_expert, n_ff, k, k_cap=0):
    """The largest M whose workspace fits trk_moe_forward_noalloc's static scratch (the need grows
    with M)."""
    lo, hi = 0, 1
    while workspace_bytes(hidden, n_expert, n_ff, k, hi, k_cap) <= NOALLOC_SCRATCH_BYTES:
        lo, hi = hi, 2 * hi
    while hi - lo > 1:
        mid = (lo + hi) // 2
        if workspace_bytes(hidden, n_expert, n_ff, k, mid, k_cap) <= NOALLOC_SCRATCH_BYTES:
            lo = mid
        else:
            hi = mid
    return lo


def forward_noalloc(hidden, n_expert, n_ff, k, w: "LayerWeights", x, out, policy=None, k_cap=0, router_dot_max_m=16,
                    hiprec=True, rlog=None, stream=None):
    """trk_moe_forward_noalloc: the layer without a context, its workspace in the library's static
    device scratch (no allocation)."""
    cfg = Cfg(hidden, n_expert, n_ff, k, 0, k_cap, router_dot_max_m, int(hiprec))
    p = C.byref(Policy(*policy)) if policy is not None else None
    check(lib().trk_moe_forward_noalloc(C.byref(cfg), p, C.byref(w.moew), _ptr(x), _ptr(rlog), x.shape[0], _ptr(out),
                                        _stream(stream)))


# ---- kernel-level wrappers (torch tensors on the GPU) ----------------------------------------

def quantize(x, kb, pair=False, stream=None):
    import torch
    m, k = (1, x.numel()) if pair else x.shape
    rows = 2 if pair else m
    q = torch.empty((rows, k), dtype=torch.int8, device=x.device)
    s = torch.empty((rows, k // kb), dtype=torch.float32, device=x.device)
    su = torch.empty((rows, k // kb), dtype=torch.int32, device=x.device)
    check(lib().trk_quantize(_ptr(x), m, k, kb, int(pair), _ptr(q), _ptr(s), _ptr(su), _stream(stream)))
    return q, s, su


def router_logits(router, x, bias=None, shexp_gate=None, gemm_order=False, stream=None):
    import torch
    m, H = x.shape
    E = router.shape[0] if router is not None else 0
    rlog = torch.empty((m, max(E, 1)), dtype=torch.float32, device=x.device)
    sh = torch.empty(m, dtype=torch.float32, device=x.device)
    check(lib().trk_router_logits(_ptr(router), _ptr(bias), _ptr(shexp_gate), _ptr(x), m, E, H, int(gemm_order),
                                  _ptr(rlog), _ptr(sh), _stream(stream)))
    return rlog[:, :E], sh


def route(logits, k, policy=None, stream=None):
    import torch
    m, E = logits.shape
    ids = torch.zeros((m, K_MAX), dtype=torch.int32, device=logits.device)
    w = torch.zeros((m, K_MAX), dtype=torch.float32, device=logits.device)
    n = torch.zeros(m, dtype=torch.int32, device=logits.device)
    p = C.byref(Policy(*policy)) if policy is not None else None
    check(lib().trk_route(_ptr(logits), m, E, k, p, _ptr(ids), _ptr(w), _ptr(n), _stream(stream)))
    return ids, w, n


def gemv(wt, rows, k, fmt, item, count, kb, q, s, su, pair=False, y=None, ldy=None, rowmap=None, accumulate=False,
         s0=0, s1=None, stream=None):
    """trk_gemv over strips [s0, s1) (all strips by default) of matrix `item` of a stack of
    `count` [rows][k] matrices in `fmt` (GGUF or TQ) held in `wt`."""
    import torch
    m = q.shape[0]
    logical = m // 2 if pair else m
    strips = (rows + 15) // 16
    s1 = strips if s1 is None else s1
    width = 16 * strips if fmt in TQ_FMTS else rows
    if y is None:
        y = torch.zeros((logical, width), dtype=torch.float32, device=q.device)
    mat = Mat(wt.data_ptr(), rows, k, fmt, count, matrix_bytes(fmt, rows, k))
    check(lib().trk_gemv(C.byref(mat), item, s0, s1, kb, _ptr(q), _ptr(s), _ptr(su), m, int(pair), _ptr(y),
                         ldy if ldy is not None else width, _ptr(rowmap), int(accumulate), _stream(stream)))
    return y


# ---- routing by scores, 8-bit products with a scale per token and per channel --------------------
#
# The kernels run on torch's current stream (or `stream`) of the current device; tensors and streams of
# others are refused.  Outputs are allocated where none is given, on the current stream as torch does: a `stream` that is not
# the current one has to wait for it before the call, as for whatever wrote the tensors given.

_torch = None  # the module, its dtypes and its device lookup once a call has needed them
_dt = None
_device = None
EXPERTS_DIRECT_M = 8  # TRK_EXPERTS_DIRECT_M


def _late():
    """torch, imported at the first call that needs it (an import statement in each call costs half a microsecond)."""
    global _torch, _dt, _device
    import torch
    _dt = {torch.float32: DT_F32, torch.bfloat16: DT_BF16, torch.float16: DT_F16}
    _device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
    _torch = torch
    return torch


def _dtype(t):
    """TRK_DT_* of a torch dtype."""
    d = _dt.get(t)
    if d is None:
        raise TrkError(f"element type {t}: float32, bfloat16 or float16 is needed")
    return d


def _u32(*values):
    """Sizes and counts as the C entry points take them; ctypes would cut what does not fit."""
    for v in values:
        if not 0 <= v < 1 << 32:
            raise TrkError(f"{v} does not fit 32 bits")


def _here(*tensors):
    """Every tensor given is on the current device."""
    dev = -1
    for t in tensors:
        if t is not None:
            at = t.get_device()
            if at < 0:
                raise TrkError("tensors have to be on the GPU")
            if dev < 0:
                dev = _device()
            if at != dev:
                raise TrkError(f"a tensor on device {at}: all have to be on the current device, {dev}")


def _stream_here(stream):
    """The hipStream_t of `stream`, which has to be one of the current device: work on another's would run there."""
    if stream is not None and stream.device_index != _device():
        raise TrkError(f"a stream of device {stream.device_index}: it has to be one of the current device, {_device()}")
    return _stream(stream)


def _rows(t, what, m=None, k=None):
    """The stride between the rows of a matrix with contiguous rows, [m][k] where they are given."""
    shape = t.shape
    if len(shape) != 2 or (m is not None and shape[0] != m) or (k is not None and shape[1] != k):
        raise TrkError(f"{what}: shape {tuple(shape)}, [{'m' if m is None else m}][{'k' if k is None else k}] is needed")
    if (shape[0] | shape[1]) >> 32:
        _u32(*shape)
    s = t.stride()
    if s[1] != 1 and shape[1] > 1:
        raise TrkError(f"{what}: the values of a row have to be contiguous")
    if shape[0] > 1:
        return s[0]
    return (shape[1] + 15) // 16 * 16  # of one row: any that the checks take


def _vector(t, what, dtype, *shape):
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise TrkError(f"{what}: a contiguous {dtype} tensor of shape {shape} is needed, not {t.dtype} {tuple(t.shape)}")


def _i8_empty(torch, rows, k, device):
    """int8 [rows][k], rows a multiple of 16 bytes apart."""
    ld = (k + 15) // 16 * 16
    q = torch.empty((rows, ld), dtype=torch.int8, device=device)
    return q if ld == k else q[:, :k]


class I8Weights:
    """A stack of int8 matrices with a scale per row (trk_i8_mat): q int8 [count][rows][k] or [rows][k], its rows and
    matrices a multiple of 16 bytes apart (`quantize_weights` makes them so), scale float32 [count][rows] or [rows].
    Keeps the tensors; copies nothing."""

    def __init__(self, q, scale):
        torch = _torch or _late()
        if q.dtype != torch.int8 or q.dim() not in (2, 3):
            raise TrkError(f"weights: int8 [count][rows][k] or [rows][k] is needed, not {q.dtype} {tuple(q.shape)}")
        _vector(scale, "weight scales", torch.float32, *q.shape[:-1])
        if min(q.shape) == 0:
            raise TrkError(f"weights: empty shape {tuple(q.shape)}")
        _u32(*q.shape)
        if q.shape[-1] > 1 and q.stride(-1) != 1:
            raise TrkError("weights: the values of a row have to be contiguous")
        _here(q, scale)
        self.q, self.scale = q, scale
        self.count = q.shape[0] if q.dim() == 3 else 1
        self.rows, self.k = q.shape[-2:]
        ld = q.stride(-2) if self.rows > 1 else (self.k + 15) // 16 * 16
        if self.k % 16:
            _whole_pieces(q, 1, 0, (q.stride(0) * (self.count - 1) if self.count > 1 else 0) + ld * (self.rows - 1) + self.k,
                          "weights")
        self.mat = I8Mat(q.data_ptr(), scale.data_ptr(), self.rows, self.k, self.count, ld,
                         q.stride(0) if self.count > 1 else 0)
        self.ref = C.byref(self.mat)
        self.device = q.get_device()


def quantize_weights(w, stream=None):
    """float [count][rows][k] or [rows][k] -> I8Weights: each row quantised as `quantize_rows` does."""
    if stream is None:
        flat = w.reshape(-1, w.shape[-1])
    else:
        with (_torch or _late()).cuda.stream(stream):  # a copy, where the rows make no one matrix: made and given back there
            flat = w.reshape(-1, w.shape[-1])
    q, s = quantize_rows(flat, stream=stream)
    q = q.as_strided((*w.shape[:-1], w.shape[-1]), (*[q.stride(0) * w.shape[-2]] * (w.dim() - 2), q.stride(0), 1))
    return I8Weights(q, s.view(w.shape[:-1]))


@functools.lru_cache(maxsize=64)
def _score_policy(*fields):
    """A trk_score_policy by reference: a program has few, and making one takes as long as a launch."""
    _u32(*fields[:5])
    return C.byref(ScorePolicy(*fields))


def route_scores(logits, k, bias=None, score="sigmoid", n_group=1, topk_group=1, group_top=2, renorm=True, factor=1.0,
                 out=None, stream=None):
    """trk_route_scores: logits [m][E] -> (ids [m][32], w [m][32], n_sel [m]); slots k .. 31 are not written."""
    torch = _torch or _late()
    if logits.dim() != 2 or logits.dtype != torch.float32 or not logits.is_contiguous():
        raise TrkError(f"logits: contiguous float32 [m][E] is needed, not {logits.dtype} {tuple(logits.shape)}")
    m, E = logits.shape
    if (m | E) >> 32:
        _u32(m, E)
    if bias is not None:
        _vector(bias, "bias", torch.float32, E)
    if score not in SCORES:
        raise TrkError(f"score {score!r}: softmax or sigmoid")
    p = _score_policy(k, SCORES[score], n_group, topk_group, group_top, int(renorm), factor)
    if out is None:
        ids = torch.empty((m, K_MAX), dtype=torch.int32, device=logits.device)
        w = logits.new_empty((m, K_MAX))
        n = ids.new_empty(m)
    else:
        ids, w, n = out
        _routing(ids, n, m, w)
    _here(logits, bias, ids, w, n)
    check(lib().trk_route_scores(logits.data_ptr(), _ptr(bias), m, E, p, ids.data_ptr(), w.data_ptr(),
                                 n.data_ptr(), _stream_here(stream)))
    return ids, w, n


def _routing(ids, n_sel, m, w=None):
    torch = _torch or _late()
    _vector(ids, "ids", torch.int32, m, K_MAX)
    _vector(n_sel, "n_sel", torch.int32, m)
    if w is not None:
        _vector(w, "w", torch.float32, m, K_MAX)


def quantize_rows(x, out=None, stream=None):
    """trk_quantize_rows: x [m][k] -> (q int8 [m][k], scale [m]); the rows of a new q are a multiple of 16 bytes apart."""
    torch = _torch or _late()
    ldx = _rows(x, "x")
    m, k = x.shape
    if out is None:
        q, scale = _i8_empty(torch, m, k, x.device), torch.empty(m, dtype=torch.float32, device=x.device)
        ldq = (k + 15) // 16 * 16
    else:
        q, scale = out
        ldq = _i8_rows(q, scale, m, k, read=False)
    _here(x, q, scale)
    check(lib().trk_quantize_rows(x.data_ptr(), _dtype(x.dtype), ldx, m, k, q.data_ptr(), ldq, scale.data_ptr(),
                                  _stream_here(stream)))
    return q, scale


def _i8_rows(q, scale, m, k, read=True):
    torch = _torch or _late()
    if q.dtype != torch.int8:
        raise TrkError(f"q: int8 is needed, not {q.dtype}")
    ld = _rows(q, "q", m, k)
    _vector(scale, "scale", torch.float32, m)
    if read and k % 16:
        _whole_pieces(q, m, ld, k, "q")
    return ld


def _whole_pieces(q, rows, ld, k, what):
    """The last row's last 16-byte piece lies inside the tensor's storage."""
    if rows and q.storage_offset() + (rows - 1) * ld + (k + 15) // 16 * 16 > q.untyped_storage().nbytes():
        raise TrkError(f"{what}: rows are read in 16-byte pieces, and the storage ends inside the last one")


def gemm_i8(w: I8Weights, q, scale, bias=None, dtype=None, out=None, accumulate=False, item=0, stream=None):
    """trk_gemm_i8: q int8 [m][k] with a scale per row, times matrix `item` of w -> [m][rows] (float32 unless `dtype` or
    `out` says otherwise)."""
    torch = _torch or _late()
    m = q.shape[0]
    if not 0 <= item < w.count:
        raise TrkError(f"item {item} out of range")
    ldq = _i8_rows(q, scale, m, w.k)
    if bias is not None:
        _vector(bias, "bias", torch.float32, w.rows)
    if out is None:
        if accumulate:
            raise TrkError("accumulate needs the output that is added to")
        out = torch.empty((m, w.rows), dtype=dtype or torch.float32, device=q.device)
        ldy = w.rows
    else:
        ldy = _rows(out, "out", m, w.rows)
    _here(q, scale, bias, out, w.q)
    check(lib().trk_gemm_i8(w.ref, item, q.data_ptr(), ldq, scale.data_ptr(), m, _ptr(bias), out.data_ptr(),
                            _dtype(out.dtype), ldy, int(accumulate), _stream_here(stream)))
    return out


@functools.lru_cache(maxsize=256)
def _plan_words(m, slots, n_expert):
    n = C.c_uint64()
    _u32(m, slots, n_expert)
    check(lib().trk_experts_plan_words(m, slots, n_expert, C.byref(n)))
    return n.value


@functools.lru_cache(maxsize=256)
def _down_work(m, slots, n_expert, rows):
    """float32 values of trk_experts_down_i8's work."""
    n = C.c_uint64()
    _u32(m, slots, n_expert, rows)
    check(lib().trk_experts_down_work_bytes(m, slots, n_expert, rows, C.byref(n)))
    return n.value // 4


def experts_plan(ids, n_sel, slots, n_expert, stream=None):
    """trk_experts_plan: the entries sorted by expert, for `experts_up_i8` and `experts_down_i8` of the same routing; None
    where the entries are so few that the products take none."""
    torch = _torch or _late()
    m = ids.shape[0]
    _routing(ids, n_sel, m)
    if m <= EXPERTS_DIRECT_M:
        return None
    words = _plan_words(m, slots, n_expert)
    _here(ids, n_sel)
    plan = torch.empty(words, dtype=torch.int32, device=ids.device)
    check(lib().trk_experts_plan(ids.data_ptr(), n_sel.data_ptr(), m, slots, n_expert, plan.data_ptr(), _stream_here(stream)))
    return plan


def _check_plan(plan, m, slots, count):
    if m <= EXPERTS_DIRECT_M:
        if slots >> 32:
            _u32(slots)
        return
    if plan is None:
        raise TrkError(f"{m} tokens of {slots} slots need a plan (experts_plan)")
    _vector(plan, "plan", _torch.int32, _plan_words(m, slots, count))


def experts_up_i8(gate: I8Weights, up: I8Weights, q, scale, ids, n_sel, slots, plan=None, dtype=None, out=None,
                  stream=None):
    """trk_experts_up_i8: q int8 [m][H] through each token's experts -> h [m * slots][F]; rows that are no entry's are not
    written."""
    torch = _torch or _late()
    m = q.shape[0]
    ldq = _i8_rows(q, scale, m, gate.k)
    _routing(ids, n_sel, m)
    _check_plan(plan, m, slots, gate.count)
    if out is None:
        out = torch.empty((m * slots, gate.rows), dtype=dtype or torch.float32, device=q.device)
        ldh = gate.rows
    else:
        ldh = _rows(out, "out", m * slots, gate.rows)
    _here(q, scale, ids, n_sel, plan, out, gate.q, up.q)
    check(lib().trk_experts_up_i8(gate.ref, up.ref, q.data_ptr(), ldq, scale.data_ptr(), m, ids.data_ptr(),
                                  n_sel.data_ptr(), slots, _ptr(plan), out.data_ptr(), _dtype(out.dtype), ldh,
                                  _stream_here(stream)))
    return out


def experts_down_i8(down: I8Weights, q, scale, ids, w, n_sel, slots, plan=None, dtype=None, out=None, work=None,
                    accumulate=False, stream=None):
    """trk_experts_down_i8: q int8 [m * slots][F] through the experts' down rows, weighted with w and summed per token ->
    [m][H].  work: at least trk_experts_down_work_bytes as a float32 tensor, allocated where it is not given."""
    torch = _torch or _late()
    m = ids.shape[0]
    ldq = _i8_rows(q, scale, m * slots, down.k)
    _routing(ids, n_sel, m, w)
    _check_plan(plan, m, slots, down.count)
    if out is None:
        if accumulate:
            raise TrkError("accumulate needs the output that is added to")
        out = torch.empty((m, down.rows), dtype=dtype or torch.float32, device=q.device)
        ldy = down.rows
    else:
        ldy = _rows(out, "out", m, down.rows)
    need = _down_work(m, slots, down.count, down.rows) if m > EXPERTS_DIRECT_M else 0
    if work is None:
        if need:
            work = torch.empty(need, dtype=torch.float32, device=q.device)
            if stream is not None:
                work.record_stream(stream)  # given back on return, while that stream still works on it
    elif work.dtype != torch.float32 or not work.is_contiguous() or work.numel() < need:
        raise TrkError(f"work: {need} contiguous float32 values are needed")
    _here(q, scale, ids, w, n_sel, plan, work, out, down.q)
    check(lib().trk_experts_down_i8(down.ref, q.data_ptr(), ldq, scale.data_ptr(), m, ids.data_ptr(), w.data_ptr(),
                                    n_sel.data_ptr(), slots, _ptr(plan), _ptr(work), out.data_ptr(), _dtype(out.dtype),
                                    ldy, int(accumulate), _stream_here(stream)))
    return out


# ---- microscaled 4-bit rows ----------------------------------------------------------------------
#
# Values uint8 [..][16 * blocks], two a byte, and scales uint8 [..][blocks], a block 32 values of a row: as the calls above in
# all else.

MX4_BLOCK = 32


def _mx4_blocks(k):
    return (k + MX4_BLOCK - 1) // MX4_BLOCK


def _mx4_rows(q, scale, m, k, what):
    """The strides between the rows of 4-bit values and of their scales, for [m][k]."""
    torch = _torch or _late()
    nb = _mx4_blocks(k)
    if q.dtype != torch.uint8 or scale.dtype != torch.uint8:
        raise TrkError(f"{what}: uint8 values and scales are needed, not {q.dtype} and {scale.dtype}")
    if q.shape != (m, 16 * nb) or scale.shape != (m, nb):
        raise TrkError(f"{what}: values [{m}][{16 * nb}] and scales [{m}][{nb}] are needed for k = {k}, not {tuple(q.shape)} "
                       f"and {tuple(scale.shape)}")
    (a, b), (c, d) = q.stride(), scale.stride()
    if b != 1 or (d != 1 and nb > 1):
        raise TrkError(f"{what}: the bytes of a row have to be contiguous")
    if m <= 1:
        a, c = 16 * nb, (nb + 3) // 4 * 4
    if nb % 4 and m:
        _whole_scales(scale, (m - 1) * c, nb, what)
    return a, c


def _whole_scales(scale, last, nb, what):
    """The last row's last 4-byte piece lies inside the tensor's storage."""
    if scale.storage_offset() + last + (nb + 3) // 4 * 4 > scale.untyped_storage().nbytes():
        raise TrkError(f"{what}: scales are read in 4-byte pieces, and the storage ends inside the last one")


class MX4Weights:
    """A stack of 4-bit matrices (trk_mx4_mat): q uint8 [count][rows][16 * blocks] or [rows][16 * blocks], its rows and matrices
    a multiple of 16 bytes apart, scale uint8 [count][rows][blocks] or [rows][blocks], a multiple of 4 (`quantize_weights_mx4`
    makes them so); k: values of a row.  Keeps the tensors; copies nothing."""

    def __init__(self, q, scale, k):
        torch = _torch or _late()
        nb = _mx4_blocks(k)
        if q.dtype != torch.uint8 or scale.dtype != torch.uint8 or q.dim() not in (2, 3):
            raise TrkError(f"weights: uint8 [count][rows][16 * blocks] or [rows][16 * blocks] and as many scales are needed, not "
                           f"{q.dtype} {tuple(q.shape)} and {scale.dtype}")
        if k < 1 or q.shape[-1] != 16 * nb or scale.shape != (*q.shape[:-1], nb):
            raise TrkError(f"weights: values [..][{16 * nb}] and scales [..][{nb}] are needed for k = {k}, not {tuple(q.shape)} and "
                           f"{tuple(scale.shape)}")
        if min(q.shape) == 0:
            raise TrkError(f"weights: empty shape {tuple(q.shape)}")
        _u32(*q.shape, k)
        if q.stride(-1) != 1 or (scale.stride(-1) != 1 and nb > 1):
            raise TrkError("weights: the bytes of a row have to be contiguous")
        _here(q, scale)
        self.q, self.scale, self.k = q, scale, k
        self.count = q.shape[0] if q.dim() == 3 else 1
        self.rows = q.shape[-2]
        many = self.count > 1
        ld, sld = (q.stride(-2), scale.stride(-2)) if self.rows > 1 else (16 * nb, (nb + 3) // 4 * 4)
        stride, sstride = (q.stride(0), scale.stride(0)) if many else (0, 0)
        if nb % 4:
            _whole_scales(scale, sstride * (self.count - 1) + sld * (self.rows - 1), nb, "weights")
        self.mat = Mx4Mat(q.data_ptr(), scale.data_ptr(), self.rows, k, self.count, ld, stride, sld, sstride)
        self.ref = C.byref(self.mat)
        self.device = q.get_device()


def quantize_mx4(x, out=None, stream=None):
    """trk_quantize_mx4: x [m][k] -> (q uint8 [m][16 * blocks], scale uint8 [m][blocks]); the scales' rows of a new pair are a
    multiple of 4 bytes apart."""
    torch = _torch or _late()
    ldx = _rows(x, "x")
    m, k = x.shape
    if out is None:
        nb = (k + 31) // 32
        ldq, lds = 16 * nb, (nb + 3) // 4 * 4
        q = torch.empty((m, ldq), dtype=torch.uint8, device=x.device)
        scale = q.new_empty((m, lds))
        if lds != nb:
            scale = scale[:, :nb]
        _here(x)
    else:
        q, scale = out
        ldq, lds = _mx4_rows(q, scale, m, k, "q")
        _here(x, q, scale)
    check(lib().trk_quantize_mx4(x.data_ptr(), _dtype(x.dtype), ldx, m, k, q.data_ptr(), ldq, scale.data_ptr(), lds,
                                 _stream_here(stream)))
    return q, scale


def dequantize_mx4(q, scale, k, dtype=None, out=None, stream=None):
    """trk_dequantize_mx4: 4-bit rows of k values -> [m][k] (float32 unless `dtype` or `out` says otherwise)."""
    torch = _torch or _late()
    m = q.shape[0]
    if (m | k) >> 32 or k < 0:
        _u32(m, k)
    ldq, lds = _mx4_rows(q, scale, m, k, "q")
    if out is None:
        out = torch.empty((m, k), dtype=dtype or torch.float32, device=q.device)
        ldy = k
    else:
        ldy = _rows(out, "out", m, k)
    _here(q, scale, out)
    check(lib().trk_dequantize_mx4(q.data_ptr(), ldq, scale.data_ptr(), lds, m, k, out.data_ptr(), _dtype(out.dtype), ldy,
                                   _stream_here(stream)))
    return out


def quantize_weights_mx4(w, stream=None):
    """float [count][rows][k] or [rows][k] -> MX4Weights: each row quantised as `quantize_mx4` does."""
    if stream is None:
        flat = w.reshape(-1, w.shape[-1])
    else:
        with (_torch or _late()).cuda.stream(stream):  # a copy, where the rows make no one matrix: made and given back there
            flat = w.reshape(-1, w.shape[-1])
    q, s = quantize_mx4(flat, stream=stream)
    lead = w.shape[:-1]

    def shaped(t):
        return t.as_strided((*lead, t.shape[1]), (*[t.stride(0) * lead[-1]] * (len(lead) - 1), t.stride(0), 1))
    return MX4Weights(shaped(q), shaped(s), w.shape[-1])


def gemm_mx4(w: MX4Weights, q, scale, bias=None, dtype=None, out=None, accumulate=False, item=0, stream=None):
    """trk_gemm_mx4: 4-bit rows [m] times matrix `item` of w -> [m][rows] (float32 unless `dtype` or `out` says otherwise)."""
    torch = _torch or _late()
    m = q.shape[0]
    if not 0 <= item < w.count:
        raise TrkError(f"item {item} out of range")
    _u32(m)
    ldq, lds = _mx4_rows(q, scale, m, w.k, "q")
    if bias is not None:
        _vector(bias, "bias", torch.float32, w.rows)
    if out is None:
        if accumulate:
            raise TrkError("accumulate needs the output that is added to")
        out = torch.empty((m, w.rows), dtype=dtype or torch.float32, device=q.device)
        ldy = w.rows
    else:
        ldy = _rows(out, "out", m, w.rows)
    _here(q, scale, bias, out, w.q)
    check(lib().trk_gemm_mx4(w.ref, item, q.data_ptr(), ldq, scale.data_ptr(), lds, m, _ptr(bias), out.data_ptr(),
                             _dtype(out.dtype), ldy, int(accumulate), _stream_here(stream)))
    return out


def experts_up_mx4(gate: MX4Weights, up: MX4Weights, q, scale, ids, n_sel, slots, plan=None, dtype=None, out=None, stream=None):
    """trk_experts_up_mx4: 4-bit rows [m] through each token's experts -> h [m * slots][F]; rows that are no entry's are not
    written."""
    torch = _torch or _late()
    m = q.shape[0]
    ldq, lds = _mx4_rows(q, scale, m, gate.k, "q")
    _routing(ids, n_sel, m)
    _check_plan(plan, m, slots, gate.count)
    if out is None:
        out = torch.empty((m * slots, gate.rows), dtype=dtype or torch.float32, device=q.device)
        ldh = gate.rows
    else:
        ldh = _rows(out, "out", m * slots, gate.rows)
    _here(q, scale, ids, n_sel, plan, out, gate.q, up.q)
    check(lib().trk_experts_up_mx4(gate.ref, up.ref, q.data_ptr(), ldq, scale.data_ptr(), lds, m, ids.data_ptr(),
                                   n_sel.data_ptr(), slots, _ptr(plan), out.data_ptr(), _dtype(out.dtype), ldh,
                                   _stream_here(stream)))
    return out


def experts_down_mx4(down: MX4Weights, q, scale, ids, w, n_sel, slots, plan=None, dtype=None, out=None, work=None,
                     accumulate=False, stream=None):
    """trk_experts_down_mx4: 4-bit rows [m * slots] through the experts' down rows, weighted with w and summed per token ->
    [m][H].  work: at least trk_experts_down_work_bytes as a float32 tensor, allocated where it is not given."""
    torch = _torch or _late()
    m = ids.shape[0]
    ldq, lds = _mx4_rows(q, scale, m * slots, down.k, "q")
    _routing(ids, n_sel, m, w)
    _check_plan(plan, m, slots, down.count)
    if out is None:
        if accumulate:
            raise TrkError("accumulate needs the output that is added to")
        out = torch.empty((m, down.rows), dtype=dtype or torch.float32, device=q.device)
        ldy = down.rows
    else:
        ldy = _rows(out, "out", m, down.rows)
    need = _down_work(m, slots, down.count, down.rows) if m > EXPERTS_DIRECT_M else 0
    work = _work_of(torch, work, need, q.device, stream)
    _here(q, scale, ids, w, n_sel, plan, work, out, down.q)
    check(lib().trk_experts_down_mx4(down.ref, q.data_ptr(), ldq, scale.data_ptr(), lds, m, ids.data_ptr(), w.data_ptr(),
                                     n_sel.data_ptr(), slots, _ptr(plan), _ptr(work), out.data_ptr(), _dtype(out.dtype), ldy,
                                     int(accumulate), _stream_here(stream)))
    return out


def _work_of(torch, work, need, device, stream):
    """`work` checked, or memory of `need` float32 values for this call."""
    if work is None:
        if need:
            work = torch.empty(need, dtype=torch.float32, device=device)
            if stream is not None:
                work.record_stream(stream)  # given back on return, while that stream still works on it
    elif work.dtype != torch.float32 or not work.is_contiguous() or work.numel() < need:
        raise TrkError(f"work: {need} contiguous float32 values are needed")
    return work


class MX4Layer:
    """A MoE layer on 4-bit experts (trk_moe_mx4_w): gate / up / down MX4Weights of the routed experts, then n_shared that every
    token takes; router float32 [E][H] (None where each call brings its logits), bias float32 [E] of the choice, shared_gate
    float32 [H].  Keeps the tensors; copies nothing."""

    def __init__(self, gate: MX4Weights, up: MX4Weights, down: MX4Weights, router=None, bias=None, n_shared=0, shared_gate=None):
        torch = _torch or _late()
        if not 0 <= n_shared < gate.count:
            raise TrkError(f"n_shared ({n_shared}) must leave routed experts of {gate.count}")
        self.n_expert, self.hidden = gate.count - n_shared, gate.k
        for t, what, shape in ((router, "router", (self.n_expert, self.hidden)), (bias, "bias", (self.n_expert,)),
                               (shared_gate, "shared_gate", (self.hidden,))):
            if t is not None:
                _vector(t, what, torch.float32, *shape)
        _here(router, bias, shared_gate, gate.q, up.q, down.q)
        self.gate, self.up, self.down, self.n_shared = gate, up, down, n_shared
        self.router, self.bias, self.shared_gate = router, bias, shared_gate
        self.w = MoeMx4W(_ptr(router), _ptr(bias), _ptr(shared_gate), gate.mat, up.mat, down.mat, n_shared)
        self.ref = C.byref(self.w)
        self._work = {}

    def work_values(self, k, m):
        """float32 values of trk_moe_mx4's work."""
        n = self._work.get((k, m))
        if n is None:
            n = C.c_uint64()
            _u32(k, m)
            check(lib().trk_moe_mx4_work_bytes(self.ref, k, m, C.byref(n)))
            n = self._work[k, m] = n.value // 4
        return n


def moe_mx4(layer: MX4Layer, x, k, rlog=None, score="sigmoid", n_group=1, topk_group=1, group_top=2, renorm=True, factor=1.0,
            dtype=None, out=None, work=None, stream=None):
    """trk_moe_mx4: x [m][H] of up to EXPERTS_DIRECT_M tokens through the layer, k experts a token chosen as `route_scores` does
    -> [m][H] (x's type unless `dtype` or `out` says otherwise).  rlog: float32 [m][E], the router's logits.  work: at least
    layer.work_values(k, m) float32 values, allocated where it is not given."""
    torch = _torch or _late()
    H = layer.hidden
    ldx = _rows(x, "x", k=H)
    m = x.shape[0]
    if rlog is not None:
        _vector(rlog, "rlog", torch.float32, m, layer.n_expert)
    elif layer.router is None:
        raise TrkError("the layer has no router: rlog is needed")
    if score not in SCORES:
        raise TrkError(f"score {score!r}: softmax or sigmoid")
    p = _score_policy(k, SCORES[score], n_group, topk_group, group_top, int(renorm), factor)
    if out is None:
        out = torch.empty((m, H), dtype=dtype or x.dtype, device=x.device)
        ldy = H
    else:
        ldy = _rows(out, "out", m, H)
    work = _work_of(torch, work, layer.work_values(k, m), x.device, stream)
    _here(x, rlog, work, out, layer.gate.q)
    check(lib().trk_moe_mx4(layer.ref, p, x.data_ptr(), _dtype(x.dtype), ldx, _ptr(rlog), m, _ptr(work), out.data_ptr(),
                            _dtype(out.dtype), ldy, _stream_here(stream)))
    return out


def swiglu(g, u, stream=None):
    import torch
    y = torch.empty_like(g)
    check(lib().trk_swiglu(_ptr(g), _ptr(u), _ptr(y), g.numel(), _stream(stream)))
    return y


def rmsnorm(x, w, eps, stream=None):
    import torch
    y = torch.empty_like(x)
    m, n = x.shape
    check(lib().trk_rmsnorm(_ptr(x), _ptr(w), eps, m, n, _ptr(y), _stream(stream)))
    return y


def gen_gguf(fmt, seed, stream_id, rows, k, dlo=1e-4, dhi=2e-3, device="cuda", stream=None):
    import torch
    out = torch.empty(rows * row_bytes(fmt, k), dtype=torch.uint8, device=device)
    check(lib().trk_gen_gguf(fmt, seed, stream_id, rows, k, dlo, dhi, _ptr(out), _stream(stream)))
    return out


def gen_normal(seed, stream_id, n, sigma=1.0, device="cuda", stream=None):
    import torch
    out = torch.empty(n, dtype=torch.float32, device=device)
    check(lib().trk_gen_normal(seed, stream_id, n, sigma, _ptr(out), _stream(stream)))
    return out


# ---- synthetic workloads ------------------------------------------------------------------------

_M64 = (1 << 64) - 1


def _mix64(z: int) -> int:
    z = (z + 0x9E3779B97F4A7C15) & _M64
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _M64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _M64
    return z ^ (z >> 31)


def rng_u64(seed: int, stream_id: int, idx: int) -> int:
    """The counter-based draw that trk_gen_gguf / trk_gen_normal use: one u64 per (seed, stream, idx)."""
    key = _mix64((seed ^ _mix64(stream_id)) & _M64)
    return _mix64((key + idx * 0xD1B54A32D192ED03) & _M64)


# Config 3's Zipf(1.1) load as a router bias.  Top-k over logits + log p (with the router's
# N(0, 0.905^2) logits) concentrates the load far beyond Zipf: only ~99 experts are touched at
# M = 512.  The load the config describes is drawing k distinct experts per token from p
# (Plackett-Luce; at M = 512, k = 10: ~460 experts touched, ~50 empty, largest group ~465, median
# 3).  zipf_bias_table.json holds the per-rank bias fitted to reproduce every rank's inclusion
# probability (make_zipf_table.py); ZIPF_BIAS_SCALE * log p is the fallback for other (E, s),
# which matches the touched and empty counts but not the largest group (~290).
ZIPF_BIAS_SCALE = 0.40
ZIPF_TABLE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "zipf_bias_table.json")


def zipf_rank_bias(E: int, s: float = 1.1):
    """The fitted per-rank bias of zipf_bias_table.json (make_zipf_table.py) when it was fitted for
    this E and s, else None."""
    import json
    import numpy as np
    try:
        with open(ZIPF_TABLE) as f:
            t = json.load(f)
    except OSError:
        return None
    if t["E"] != E or abs(t["s"] - s) > 1e-12:
        return None
    return np.array(t["bias"], np.float64)


def zipf_bias(seed: int, E: int, s: float = 1.1, scale: float = None, stream_id: int = 5):
    """Router bias for config 3's Zipf(s) load, over the permutation pi that sorts
    rng_u64(seed, stream_id, e): the expert of rank j gets b_j (float32 numpy array of E).

    b_j is the fitted per-rank bias of zipf_bias_table.json when one exists for (E, s): top-10
    over the synthetic router's N(0, 0.905^2) logits plus b then includes each expert as often as
    drawing 10 distinct experts per token from Zipf(s) does (make_zipf_table.py).  Otherwise, or
    with an explicit scale, b_j = scale * log p_j with p_j ~ j^-s (scale 0.40 by default)."""
    import numpy as np
    keys = np.array([rng_u64(seed, stream_id, e) for e in range(E)], np.uint64)
    perm = np.argsort(keys, kind="stable")  # perm[j] = the expert of rank j
    rank_b = zipf_rank_bias(E, s) if scale is None else None
    if rank_b is None:
        p = 1.0 / np.arange(1, E + 1, dtype=np.float64) ** s
        p /= p.sum()
        rank_b = (ZIPF_BIAS_SCALE if scale is None else scale) * np.log(p)
    b = np.zeros(E, np.float32)
    b[perm] = rank_b.astype(np.float32)
    return b
