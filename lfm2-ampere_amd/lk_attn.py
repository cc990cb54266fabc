"""Python host mirror of the attention entry points (ctypes over liblk_attn.so).

The reference engine is C++ and launches its attention kernels directly
(/root/reference/src/engine.cu:638-641 for decode, :1082-1089 and :1122 for
prefill).  This module binds the C ABI of ``include/lk_attn.h`` under the
reference's kernel names (``attn_split`` for ``k_attn_split`` and so on) so
tests and the benchmark read like the reference's own harnesses.  PyTorch is
used only to own device memory and streams; every computation runs in the HIP
library.  There is no fallback: if the library is missing or fails, calls raise.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional, Sequence

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "liblk_attn.so")

N_HEADS, N_KV_HEADS, HEAD_DIM = 32, 8, 64
PARTW = 4 + HEAD_DIM
DECODE_MAX_SEQ = 8192
Q8_1_BYTES = 36

# Every symbol the header declares; tests check the library exports them all.
EXPORTS = (
    "lk_attn_config", "lk_attn_part_bytes", "lk_last_error",
    "lk_attn_split", "lk_attn_combine", "lk_attn_decode", "lk_attention_decode",
    "lk_decode_graph_create", "lk_decode_graph_launch", "lk_decode_graph_nodes",
    "lk_decode_graph_destroy",
    "lk_pf_q8", "lk_pf_k8", "lk_pf_kmean", "lk_pf_attn8", "lk_pf_attn", "lk_pf_split_override", "lk_pf_pair_override",
    "lk_pf_qk_i32", "lk_pf_plan_items", "lk_read_probe", "lk_qk_norm_rope", "lk_pf_qknr",
    "lk_decode_step_graph_create", "lk_decode_graph_run",
    "lk_pf_ctx_create", "lk_pf_ctx_destroy", "lk_pf_chunk_attn", "lk_pf_chunk_done", "lk_pf_ctx_buffers",
    "lk_pf_attn8_q81", "lk_pf_attn_q81", "lk_pf_quant_rows", "lk_gemv_q4_0", "lk_pf_gemm_q4_0",
    "lk_attn_decode_noalloc", "lk_rope_freq_table",
    "lk_pf_part_bytes", "lk_pf_attn8_ws", "lk_pf_attn_ws", "lk_pf_gsync_limit", "lk_pf_gsync_faults",
    "lk_synth_f32", "lk_norm_q8", "lk_gemm_i8",
    "lk_moe_work_bytes", "lk_moe_q4_0",
    "lk_paged_append", "lk_paged_attn_work_bytes", "lk_paged_attn", "lk_paged_commit",
)


class LkError(RuntimeError):
    """A C-ABI call returned a non-zero hipError_t."""


_lib: Optional[ctypes.CDLL] = None
_raw_stream = _device = None                # torch's current raw stream and device, bound by load()


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load liblk_attn.so (raises if it has not been built)."""
    global _lib, _raw_stream, _device
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise FileNotFoundError(
            f"{path} is missing: build it with `make -C lfm2-ampere_amd` "
            "(or __graft_entry__.build()); there is no fallback path")
    # torch (whose tensors this module passes as device memory) carries its own
    # HIP runtime under the same soname; load it first so the process has one
    # runtime and torch's streams and allocations are valid for the library.
    import torch
    # (absent from a CPU-only torch, where the host-side entry points still work)
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    _device = getattr(torch._C, "_cuda_getDevice", None)
    lib = ctypes.CDLL(path)
    P, I, S = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
    sig = {
        "lk_attn_config": ([P, P, P], I),
        "lk_attn_part_bytes": ([], S),
        "lk_rope_freq_table": ([P], I),
        "lk_last_error": ([], ctypes.c_char_p),
        "lk_attn_split": ([P, P, P, P, P, P], I),
        "lk_attn_combine": ([P, P, P, P, P], I),
        "lk_attn_decode": ([P, P, P, P, P, P, P, P], I),
        "lk_attn_decode_noalloc": ([P, P, P, P, P, P, P], I),
        "lk_attention_decode": ([P, P, P, P, P, P, P], I),
        "lk_decode_graph_create": ([I, P, P, P, P, P, P, P, P, P], I),
        "lk_decode_graph_launch": ([P, P], I),
        "lk_decode_graph_nodes": ([P, P], I),
        "lk_decode_graph_destroy": ([P], I),
        "lk_pf_q8": ([P, I, P, P, P, P, P], I),
        "lk_pf_k8": ([P, I, I, P, I, P, P, P], I),
        "lk_pf_kmean": ([P, I, P, P], I),
        "lk_pf_attn8": ([P, P, P, P, I, I, P, P, I, P, P, I, I, P, P], I),
        "lk_pf_attn": ([P, I, I, P, P, P, P], I),
        "lk_pf_split_override": ([I], I),
        "lk_pf_pair_override": ([I], I),
        "lk_pf_qk_i32": ([P, I, P, I, P, P], I),
        "lk_pf_plan_items": ([I, I, I, I, I, P, I], I),
        "lk_read_probe": ([P, S, P, P], I),
        "lk_gemv_q4_0": ([P, P, P, I, I, P, I, P, ctypes.c_float, P], I),
        "lk_pf_gemm_q4_0": ([P, P, I, I, P, P, I, P, P, I, I, P], I),
        "lk_qk_norm_rope": ([P, P, P, P, P, P, P, P, P], I),
        "lk_pf_qknr": ([P, P, P, I, I, P, P, P, P, P, I, P, P], I),
        "lk_decode_step_graph_create": ([I, P, P, P, P, P], I),
        "lk_decode_graph_run": ([P, I, P], I),
        "lk_pf_ctx_create": ([I, I, I, I, I, I, I, P], I),
        "lk_pf_ctx_destroy": ([P], I),
        "lk_pf_chunk_attn": ([P, I, P, P, P, I, I, P, P, P, P, P, P], I),
        "lk_pf_attn8_q81": ([P, P, P, P, I, I, P, P, I, P, P, I, I, P, P, P, P], I),
        "lk_pf_attn_q81": ([P, I, I, P, P, P, P, P, P], I),
        "lk_pf_quant_rows": ([P, I, I, I, P, P, P], I),
        "lk_pf_chunk_done": ([P, I], I),
        "lk_pf_ctx_buffers": ([P, I, P, P, P, P, P, P], I),
        "lk_pf_part_bytes": ([], S),
        "lk_pf_attn8_ws": ([P, P, P, P, I, I, P, P, I, P, P, I, I, P, P, P, P, S, P], I),
        "lk_pf_attn_ws": ([P, I, I, P, P, P, P, P, P, S, P], I),
        "lk_pf_gsync_limit": ([I], I),
        "lk_pf_gsync_faults": ([P, I], I),
        "lk_synth_f32": ([I, ctypes.c_uint64, S, ctypes.c_float, ctypes.c_float, P, P], I),
        "lk_norm_q8": ([I, P, I, P, I, P, ctypes.c_float, I, I, P, I, P, I, I, P, I, P, P], I),
        "lk_moe_work_bytes": ([P, I], S),
        "lk_moe_q4_0": ([P, I, P, I, I, P, I, P, I, P, P, P, S, P], I),
        "lk_gemm_i8": ([P, I, P, P, I, P, I, I, I, I, P, I, P, I, P], I),
        "lk_paged_append": ([P, P, I, P, I, P, I, P, I, P, P, ctypes.c_float, P, I, I, P, I, P], I),
        "lk_paged_attn_work_bytes": ([P, I, I], S),
        "lk_paged_attn": ([P, P, I, P, I, ctypes.c_float, ctypes.c_float, P, P, I, P, S, P], I),
        "lk_paged_commit": ([P, P, P, I, P, P, P], I),
    }
    for name, (args, res) in sig.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = res
    _lib = lib
    return lib


def _check(rc: int, what: str) -> None:
    if rc != 0:
        msg = load().lk_last_error().decode(errors="replace")
        raise LkError(f"{what} failed (hipError {rc}): {msg}")


def _ptr(t) -> Optional[int]:
    """Device pointer of a tensor (None -> NULL).  Checks residency and layout."""
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("lk_attn: tensors must live in device memory")
    if not t.is_contiguous():
        raise ValueError("lk_attn: tensors must be contiguous")
    return t.data_ptr()


def _stream(stream) -> Optional[int]:
    """hipStream_t of `stream`, or of torch's current stream.  The raw handle is
    read directly: torch.cuda.current_stream() builds a Stream object, 2.7 us of
    a host path that is otherwise 8 us for a decode call (two launches)."""
    if stream is None:
        if _raw_stream is None or _device is None:
            import torch
            return torch.cuda.current_stream().cuda_stream or None
        return _raw_stream(_device()) or None
    return stream.cuda_stream or None


def config() -> dict:
    a, b, c = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    _check(load().lk_attn_config(ctypes.byref(a), ctypes.byref(b), ctypes.byref(c)), "lk_attn_config")
    return {"split_cap": a.value, "target_n": b.value, "split_min": c.value}


def part_bytes() -> int:
    return int(load().lk_attn_part_bytes())


def attn_slices(seq: int) -> tuple:
    """The library's split-K slice rule (reference kernels.cuh:630-635)."""
    c = config()
    s = (seq + c["target_n"] - 1) // c["target_n"]
    s = max(c["split_min"], min(c["split_cap"], s))
    return s, (seq + s - 1) // s


# ---- decode (reference kernels.cuh:644-658) -------------------------------------
def attn_split(q, kc, vc, d_pos, part, stream=None) -> None:
    _check(load().lk_attn_split(_ptr(q), _ptr(kc), _ptr(vc), _ptr(d_pos), _ptr(part),
                                _stream(stream)), "lk_attn_split")


def attn_combine(part, d_pos, out=None, yq8=None, stream=None) -> None:
    _check(load().lk_attn_combine(_ptr(part), _ptr(d_pos), _ptr(out), _ptr(yq8),
                                  _stream(stream)), "lk_attn_combine")


def attn_decode(q, kc, vc, d_pos, part, out=None, yq8=None, stream=None) -> None:
    _check(load().lk_attn_decode(_ptr(q), _ptr(kc), _ptr(vc), _ptr(d_pos), _ptr(part),
                                 _ptr(out), _ptr(yq8), _stream(stream)), "lk_attn_decode")


def attn_decode_noalloc(q, kc, vc, d_pos, out=None, yq8=None, stream=None) -> None:
    """lk_attn_decode without a `part` workspace: the library's static
    per-device scratch holds the partials (calls overlapping on one GPU race)."""
    _check(load().lk_attn_decode_noalloc(_ptr(q), _ptr(kc), _ptr(vc), _ptr(d_pos),
                                         _ptr(out), _ptr(yq8), _stream(stream)), "lk_attn_decode_noalloc")


def attention_decode(q, kc, vc, d_pos, out=None, yq8=None, stream=None) -> None:
    _check(load().lk_attention_decode(_ptr(q), _ptr(kc), _ptr(vc), _ptr(d_pos), _ptr(out),
                                      _ptr(yq8), _stream(stream)), "lk_attention_decode")


class DecodeLayer(ctypes.Structure):
    """lk_decode_layer (include/lk_attn.h): one layer's buffers for the step graph."""
    _fields_ = [(n, ctypes.c_void_p) for n in
                ("q_src", "k_src", "v_src", "q", "k", "q_norm", "k_norm", "kc", "vc", "out", "yq8",
                 "wo_qs", "wo_d", "x")]


class DecodeStepGraph:
    """The decode step's attention slice (per layer: qk norm + RoPE of the
    projection rows + cache append, split, combine; then d_pos += 1) captured
    into one hipGraph; run(n) replays it n times."""

    def __init__(self, layers: Sequence[dict], d_pos, part, stream=None):
        import torch
        n = len(layers)
        arr = (DecodeLayer * n)()
        for i, L in enumerate(layers):
            for f, _ in DecodeLayer._fields_:
                setattr(arr[i], f, _ptr(L.get(f)))
        self._keep = (layers, d_pos, part, arr)
        self._stream = stream if stream is not None else torch.cuda.Stream()
        h = ctypes.c_void_p()
        _check(load().lk_decode_step_graph_create(n, arr, _ptr(d_pos), _ptr(part),
                                                  self._stream.cuda_stream, ctypes.byref(h)),
               "lk_decode_step_graph_create")
        self._h = h

    @property
    def stream(self):
        return self._stream

    def nodes(self) -> int:
        n = ctypes.c_size_t()
        _check(load().lk_decode_graph_nodes(self._h, ctypes.byref(n)), "lk_decode_graph_nodes")
        return n.value

    def run(self, n_steps: int = 1) -> None:
        _check(load().lk_decode_graph_run(self._h, int(n_steps), self._stream.cuda_stream), "lk_decode_graph_run")

    def close(self) -> None:
        if getattr(self, "_h", None):
            load().lk_decode_graph_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class DecodeGraph:
    """n_layers x (split, combine) captured into one hipGraph."""

    def __init__(self, qs: Sequence, kcs: Sequence, vcs: Sequence, d_pos, part,
                 outs: Optional[Sequence] = None, yq8s: Optional[Sequence] = None, stream=None):
        import torch
        n = len(qs)
        if not (len(kcs) == n and len(vcs) == n):
            raise ValueError("DecodeGraph: per-layer lists must have equal length")
        arr = ctypes.c_void_p * n
        self._keep = (qs, kcs, vcs, d_pos, part, outs, yq8s)
        self._stream = stream if stream is not None else torch.cuda.Stream()
        h = ctypes.c_void_p()
        o = arr(*[_ptr(t) for t in outs]) if outs is not None else None
        y = arr(*[_ptr(t) for t in yq8s]) if yq8s is not None else None
        _check(load().lk_decode_graph_create(
            n, arr(*[_ptr(t) for t in qs]), arr(*[_ptr(t) for t in kcs]),
            arr(*[_ptr(t) for t in vcs]), _ptr(d_pos), _ptr(part), o, y,
            self._stream.cuda_stream, ctypes.byref(h)), "lk_decode_graph_create")
        self._h = h

    @property
    def stream(self):
        return self._stream

    def nodes(self) -> int:
        n = ctypes.c_size_t()
        _check(load().lk_decode_graph_nodes(self._h, ctypes.byref(n)), "lk_decode_graph_nodes")
        return n.value

    def launch(self) -> None:
        _check(load().lk_decode_graph_launch(self._h, self._stream.cuda_stream), "lk_decode_graph_launch")

    def close(self) -> None:
        if getattr(self, "_h", None):
            load().lk_decode_graph_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- prefill (reference prefill.cuh:85-109) -------------------------------------
def pf_q8(qh, m, cm, q8, qsc, qcs, stream=None) -> None:
    _check(load().lk_pf_q8(_ptr(qh), m, _ptr(cm), _ptr(q8), _ptr(qsc), _ptr(qcs), _stream(stream)),
           "lk_pf_q8")


def pf_k8(kc, p0, p1, cm, kstride, k8, ksc, stream=None) -> None:
    _check(load().lk_pf_k8(_ptr(kc), p0, p1, _ptr(cm), kstride, _ptr(k8), _ptr(ksc), _stream(stream)),
           "lk_pf_k8")


def pf_kmean(kc, n, cm, stream=None) -> None:
    _check(load().lk_pf_kmean(_ptr(kc), n, _ptr(cm), _stream(stream)), "lk_pf_kmean")


def pf_attn8(q8, qsc, qcs, qh, m, P, k8, ksc, kstride, kc, vc, near, sink, o, stream=None) -> None:
    """Int8-scored prefill attention (reference k_pf_attn8).  q8, qsc and qcs
    None: the kernel quantises qh itself (lk_pf_q8's arithmetic, no
    smoothing), with the same output as the two-kernel path."""
    _check(load().lk_pf_attn8(_ptr(q8), _ptr(qsc), _ptr(qcs), _ptr(qh), m, P, _ptr(k8), _ptr(ksc),
                              kstride, _ptr(kc), _ptr(vc), near, sink, _ptr(o), _stream(stream)),
           "lk_pf_attn8")


def pf_attn(qh, m, P, kc, vc, o, stream=None) -> None:
    _check(load().lk_pf_attn(_ptr(qh), m, P, _ptr(kc), _ptr(vc), _ptr(o), _stream(stream)), "lk_pf_attn")


def pf_attn8_q81(q8, qsc, qcs, qh, m, P, k8, ksc, kstride, kc, vc, near, sink, o, aqs, asc, stream=None) -> None:
    _check(load().lk_pf_attn8_q81(_ptr(q8), _ptr(qsc), _ptr(qcs), _ptr(qh), int(m), int(P), _ptr(k8), _ptr(ksc),
                                  int(kstride), _ptr(kc), _ptr(vc), int(near), int(sink), _ptr(o), _ptr(aqs),
                                  _ptr(asc), _stream(stream)), "lk_pf_attn8_q81")


def pf_attn_q81(qh, m, P, kc, vc, o, aqs, asc, stream=None) -> None:
    _check(load().lk_pf_attn_q81(_ptr(qh), int(m), int(P), _ptr(kc), _ptr(vc), _ptr(o), _ptr(aqs), _ptr(asc),
                                 _stream(stream)), "lk_pf_attn_q81")


def pf_part_bytes() -> int:
    """Bytes of the largest split-K partial workspace a prefill launch uses."""
    return int(load().lk_pf_part_bytes())


def _nbytes(t) -> int:
    return 0 if t is None else t.numel() * t.element_size()


def pf_attn8_ws(q8, qsc, qcs, qh, m, P, k8, ksc, kstride, kc, vc, near, sink, o, aqs, asc, work,
                stream=None) -> None:
    """pf_attn8_q81 with a caller-owned split-K workspace (a device tensor; None:
    the library's static scratch)."""
    _check(load().lk_pf_attn8_ws(_ptr(q8), _ptr(qsc), _ptr(qcs), _ptr(qh), int(m), int(P), _ptr(k8), _ptr(ksc),
                                 int(kstride), _ptr(kc), _ptr(vc), int(near), int(sink), _ptr(o), _ptr(aqs),
                                 _ptr(asc), _ptr(work), _nbytes(work), _stream(stream)), "lk_pf_attn8_ws")


def pf_attn_ws(qh, m, P, kc, vc, o, aqs, asc, work, stream=None) -> None:
    _check(load().lk_pf_attn_ws(_ptr(qh), int(m), int(P), _ptr(kc), _ptr(vc), _ptr(o), _ptr(aqs), _ptr(asc),
                                _ptr(work), _nbytes(work), _stream(stream)), "lk_pf_attn_ws")


def pf_gsync_limit(polls: int) -> None:
    """Poll bound of the paired prefill kernel's group barriers (0: default)."""
    _check(load().lk_pf_gsync_limit(int(polls)), "lk_pf_gsync_limit")


def pf_gsync_faults(reset: bool = False) -> int:
    """Group barriers that gave up on this device since the last reset (synchronous)."""
    c = ctypes.c_uint()
    _check(load().lk_pf_gsync_faults(ctypes.byref(c), int(bool(reset))), "lk_pf_gsync_faults")
    return c.value


SYNTH_NORMAL, SYNTH_UNIFORM, SYNTH_STUDENT4 = 0, 1, 2


def synth(kind: int, seed: int, out, lo: float = 0.0, hi: float = 1.0, stream=None) -> None:
    """Fill the fp32 device tensor `out` with the seeded splitmix64 stream of
    `seed` (kind: SYNTH_NORMAL, SYNTH_UNIFORM in [lo, hi), SYNTH_STUDENT4)."""
    if out.dtype != __import__("torch").float32:
        raise ValueError("synth: out must be fp32")
    _check(load().lk_synth_f32(int(kind), int(seed) & ((1 << 64) - 1), out.numel(), float(lo), float(hi),
                               _ptr(out), _stream(stream)), "lk_synth_f32")


def pf_quant_rows(X, rows, ld, kb, qs, sc, stream=None) -> None:
    _check(load().lk_pf_quant_rows(_ptr(X), int(rows), int(ld), int(kb), _ptr(qs), _ptr(sc), _stream(stream)),
           "lk_pf_quant_rows")


def pf_pair_override(mode: int) -> None:
    """Paired prefill workgroups (blocks i and nq-1-i in one launch unit):
    -1 never, 0 automatic, 1 whenever the chunk has at least two 64-row blocks."""
    _check(load().lk_pf_pair_override(int(mode)), "lk_pf_pair_override")


def pf_split_override(tiles: int) -> None:
    """-1 never split prefill blocks, 0 automatic, n > 0 parts of <= n key tiles."""
    _check(load().lk_pf_split_override(int(tiles)), "lk_pf_split_override")


def read_probe(buf, sink, stream=None) -> None:
    """Plain streaming read of a device tensor (measurement reference)."""
    _check(load().lk_read_probe(_ptr(buf), buf.numel() * buf.element_size(), _ptr(sink),
                                _stream(stream)), "lk_read_probe")


def gemv_q4_0(qs, d, xq, out_rows: int, bpr: int, y, add_residual: bool = False, ssq=None,
              eps: float = 1e-5, stream=None) -> None:
    """Q4_0 x Q8_1 GEMV (reference k_gemv_q4_0): qs [out_rows][bpr] 16-byte
    blocks, d fp16 [out_rows][bpr], xq [bpr] Q8_1 blocks (36 bytes), y fp32
    [out_rows] (accumulated into when add_residual); ssq: 64 fp32 norm partials
    or None."""
    _check(load().lk_gemv_q4_0(_ptr(qs), _ptr(d), _ptr(xq), int(out_rows), int(bpr), _ptr(y),
                               int(bool(add_residual)), _ptr(ssq), float(eps), _stream(stream)),
           "lk_gemv_q4_0")


def pf_gemm_q4_0(qs, d, N: int, bpr: int, aqs, asc, ntok: int, out, out_ld: int = None,
                 add: bool = False, scale=None, stream=None) -> None:
    """Q4_0 x planar Q8_1 GEMM of a prefill chunk (reference pf_gemm_dense, one
    tensor, plain epilogue): out[t][r] (+)= scale[t] * W[r] . x[t]."""
    _check(load().lk_pf_gemm_q4_0(_ptr(qs), _ptr(d), int(N), int(bpr), _ptr(aqs), _ptr(asc), int(ntok),
                                  _ptr(scale), _ptr(out), int(N if out_ld is None else out_ld),
                                  int(bool(add)), _stream(stream)), "lk_pf_gemm_q4_0")


def pf_plan_items(m: int, P: int, near: int, sink: int, int8: bool = True, max_items: int = 1024):
    """The split work list of a prefill chunk, in dispatch order: a list of
    (query block, first key tile, end key tile, partial slot or -1); [] for an
    unsplit launch.  Host-side only."""
    import ctypes
    buf = (ctypes.c_int32 * (4 * max_items))()
    n = load().lk_pf_plan_items(int(m), int(P), int(near), int(sink), int(bool(int8)),
                                ctypes.addressof(buf), int(max_items))
    if n < 0:
        raise LkError("lk_pf_plan_items: bad arguments")
    return [tuple(buf[4 * i:4 * i + 4]) for i in range(min(n, max_items))]


def pf_qk_i32(q8, m, k8, n, s, stream=None) -> None:
    _check(load().lk_pf_qk_i32(_ptr(q8), m, _ptr(k8), n, _ptr(s), _stream(stream)), "lk_pf_qk_i32")


def kstride_for(S: int) -> int:
    """ksc row stride for S positions: rounded up to 4 (reference engine.cu:979)."""
    return (S + 3) & ~3


# ---- attention-input producers (reference kernels.cu:871-915, prefill.cu:975-1016) ----
def qk_norm_rope(qf, kf, vf, qn, kn, d_pos, kc, vc, stream=None) -> None:
    _check(load().lk_qk_norm_rope(_ptr(qf), _ptr(kf), _ptr(vf), _ptr(qn), _ptr(kn), _ptr(d_pos),
                                  _ptr(kc), _ptr(vc), _stream(stream)), "lk_qk_norm_rope")


def pf_qknr(Y, qn, kn, m, P, qh, kc, vc, k8=None, ksc=None, kstride=0, cm=None, stream=None) -> None:
    _check(load().lk_pf_qknr(_ptr(Y), _ptr(qn), _ptr(kn), int(m), int(P), _ptr(qh), _ptr(kc), _ptr(vc),
                             _ptr(k8), _ptr(ksc), int(kstride), _ptr(cm), _stream(stream)), "lk_pf_qknr")


# ---- the 8-bit feed-forward half -------------------------------------------------
# These check types, shapes and devices themselves (rows may be strided views),
# and enqueue on the tensors' device, whichever is current: on its current stream,
# or on `stream`, which must be one of that device.
F32, F16, BF16 = 0, 1, 2
Q8_ROW, Q81_PLANAR, Q81_BLOCK = 0, 1, 2
_torch = _types = None                      # torch; its dtype -> LK_F32 / LK_F16 / LK_BF16


def _type_of(t, what: str) -> int:
    global _torch, _types
    if _types is None:
        import torch
        _torch, _types = torch, {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
    ty = _types.get(t.dtype)
    if ty is None:
        raise ValueError(f"{what}: fp32, fp16 or bf16 rows, not {t.dtype}")
    return ty


def _rows2(t, shape: tuple, dtype, dev: int, what: str) -> tuple:
    """(pointer, row stride) of a [rows][n] tensor of a dtype on device `dev` whose
    rows are contiguous; (None, 0) for None."""
    if t is None:
        return None, 0
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{what}: {dtype} {list(shape)} wanted, not {t.dtype} {list(t.shape)}")
    if t.get_device() != dev:
        raise ValueError(f"{what}: on another device, or not in device memory")
    rows, n = shape
    s0, s1 = t.stride()
    if (s1 != 1 and n > 1) or (rows > 1 and s0 < n):
        raise ValueError(f"{what}: rows must be contiguous and must not overlap (strides {s0}, {s1})")
    if s0 > 0x7FFFFFFF and rows > 1 or rows > 0x7FFFFFFF or n > 0x7FFFFFFF:
        raise ValueError(f"{what}: {rows} rows of {n}, {s0} apart: beyond what the entry points count")
    return t.data_ptr(), s0 if rows > 1 else n


def _flat(t, shape: tuple, dtype, dev: int, what: str):
    """Pointer of a contiguous tensor of a shape and dtype on device `dev`."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what}: contiguous {dtype} {list(shape)} on the rows' device wanted, not {t.dtype} "
                         f"{list(t.shape)}")
    return t.data_ptr()


def _on(dev: int, stream, call, *args) -> int:
    """call(*args, stream) with `dev` as the current device: the given stream, or
    the device's current one."""
    if dev < 0:
        raise ValueError("lk_attn: tensors must live in device memory")
    if stream is not None and getattr(stream, "device_index", dev) != dev:
        raise ValueError("lk_attn: the stream is one of another device than the tensors'")
    if _raw_stream is not None and _device is not None and _device() == dev:
        return call(*args, (_raw_stream(dev) if stream is None else stream.cuda_stream) or None)
    import torch
    with torch.cuda.device(dev):
        return call(*args, (torch.cuda.current_stream() if stream is None else stream).cuda_stream or None)


def norm_q8(x, w, q, sc=None, delta=None, res=None, y=None, eps: float = 1e-5, stream=None) -> None:
    """h = x + delta, y = rmsnorm(h) * w, and y in 8 bits, in one pass over the
    rows [rows][n] of fp32, fp16 or bf16 (lk_norm_q8).  `res` takes h (it may be x or
    delta), `y` the normed rows, both of x's type.  The 8-bit form follows from the outputs:
      sc fp32 [rows], q int8 [rows][n]                    a scale a row (gemm_i8)
      sc fp32 [rows][n/32][2], q int8 [rows][n]           planar Q8_1 (pf_gemm_q4_0)
      sc None, q uint8 [rows][n/32 * 36]                  Q8_1 blocks (gemv_q4_0)"""
    lib = _lib or load()
    ty = _type_of(x, "norm_q8")
    if x.dim() != 2:
        raise ValueError("norm_q8: x must be [rows, n]")
    shape = rows, n = x.shape
    dev = x.get_device()
    px, ldx = _rows2(x, shape, x.dtype, dev, "norm_q8: x")
    pd, ldd = _rows2(delta, shape, x.dtype, dev, "norm_q8: delta")
    pr, ldr = _rows2(res, shape, x.dtype, dev, "norm_q8: res")
    py, ldy = _rows2(y, shape, x.dtype, dev, "norm_q8: y")
    pw = _flat(w, (n,), _torch.float32, dev, "norm_q8: w")
    if sc is None:
        form, ldq, ps = Q81_BLOCK, n, None
        pq = _flat(q, (rows, n // 32 * Q8_1_BYTES), _torch.uint8, dev, "norm_q8: q")
    elif sc.dim() == 1:
        form, ps = Q8_ROW, _flat(sc, (rows,), _torch.float32, dev, "norm_q8: sc")
        pq, ldq = _rows2(q, shape, _torch.int8, dev, "norm_q8: q")
    else:
        form, ldq, ps = Q81_PLANAR, n, _flat(sc, (rows, n // 32, 2), _torch.float32, dev, "norm_q8: sc")
        pq = _flat(q, shape, _torch.int8, dev, "norm_q8: q")
    rc = _on(dev, stream, lib.lk_norm_q8, ty, px, ldx, pd, ldd, pw, eps, rows, n, pr, ldr, py, ldy, form, pq, ldq, ps)
    if rc:
        _check(rc, "lk_norm_q8")


def i8_rows(rows: int, n: int, device="cuda"):
    """An int8 [rows][n] tensor whose rows lie a multiple of 16 bytes apart, as
    gemm_i8 takes them (zeroed)."""
    import torch
    return torch.zeros(rows, (n + 15) // 16 * 16, dtype=torch.int8, device=device)[:, :n]


def _padded(t, ld: int, what: str) -> int:
    """Row stride of int8 rows of which the last, too, has readable bytes up to
    the next multiple of 16 (a single row has no stride of its own)."""
    rows, n = t.shape
    if rows == 1:
        ld = n + 15 & ~15
    end = t.storage_offset() + (rows - 1) * ld + (n + 15 & ~15)
    if rows and end > t.untyped_storage().nbytes():
        raise ValueError(f"{what}: the last row's bytes up to a multiple of 16 lie past its storage (see i8_rows)")
    return ld


def gemm_i8(x, sx, w, sw, out, res=None, stream=None) -> None:
    """out[t][r] = (res[t][r] +) (x[t] . w[r]) * sx[t] * sw[r] (lk_gemm_i8): x int8
    [M][K] and w int8 [N][K] with rows a multiple of 16 bytes apart (i8_rows), sx fp32
    [M], sw fp32 [N], out (and res, which may be out) fp32, fp16 or bf16 [M][N]."""
    lib = _lib or load()
    ty = _type_of(out, "gemm_i8")
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError("gemm_i8: x must be [M, K] and w [N, K]")
    M, K = x.shape
    N = w.shape[0]
    dev = x.get_device()
    px, ldx = _rows2(x, x.shape, _torch.int8, dev, "gemm_i8: x")
    pw, ldw = _rows2(w, (N, K), _torch.int8, dev, "gemm_i8: w")
    po, ldo = _rows2(out, (M, N), out.dtype, dev, "gemm_i8: out")
    pr, ldr = _rows2(res, (M, N), out.dtype, dev, "gemm_i8: res")
    if K % 16:
        ldx, ldw = _padded(x, ldx, "gemm_i8: x"), _padded(w, ldw, "gemm_i8: w")
    rc = _on(dev, stream, lib.lk_gemm_i8, px, ldx, _flat(sx, (M,), _torch.float32, dev, "gemm_i8: sx"), pw, ldw,
             _flat(sw, (N,), _torch.float32, dev, "gemm_i8: sw"), M, N, K, ty, pr, ldr, po, ldo)
    if rc:
        _check(rc, "lk_gemm_i8")


class MoeDesc(ctypes.Structure):
    """lk_moe (include/lk_attn.h)."""
    _fields_ = [(n, ctypes.c_int) for n in ("n_experts", "top_k", "hidden", "ffn", "score", "renorm")] + \
        [("scale", ctypes.c_float)] + \
        [(n, ctypes.c_void_p) for n in ("router", "bias", "gate_qs", "gate_d", "up_qs", "up_d", "down_qs", "down_d")]


class MoeQ4_0:
    """A mixture-of-experts layer of Q4_0 experts for up to `max_tokens` tokens a
    call (lk_moe_q4_0): router fp32 [E][hidden]; gate and up pairs (qs uint8
    [E][ffn][hidden/32][16], d fp16 [E][ffn][hidden/32]), down the same as
    [E][hidden][ffn/32]; score "sigmoid" or "softmax", bias fp32 [E] for the choice
    only.  Keeps the weights and one workspace: calls on it must be ordered (one
    stream, or events); calls that may overlap, captured graphs among them, are given
    workspaces of their own (`work`, uint8 of work_bytes()).  A layer may be dropped while
    streams still work on it, as far as its workspace goes (Tensor.record_stream; the weights are
    the caller's tensors); a captured graph needs its layer as long as it is replayed."""

    def __init__(self, router, gate, up, down, top_k: int, score: str = "sigmoid", bias=None, renorm: bool = True,
                 scale: float = 1.0, max_tokens: int = 64):
        import torch
        if score not in ("sigmoid", "softmax"):
            raise ValueError(f"MoeQ4_0: score {score!r}")
        if router.dim() != 2 or gate[0].dim() != 4:
            raise ValueError("MoeQ4_0: router must be [E, hidden], quants [E, rows, blocks, 16]")
        dev, (E, hidden), ffn = router.get_device(), router.shape, gate[0].shape[1]
        if hidden % 32 or ffn % 32 or hidden < 32 or ffn < 32:
            raise ValueError(f"MoeQ4_0: hidden {hidden}, ffn {ffn} must be multiples of 32")
        ptr = [_flat(router, (E, hidden), torch.float32, dev, "MoeQ4_0: router"),
               None if bias is None else _flat(bias, (E,), torch.float32, dev, "MoeQ4_0: bias")]
        for what, (qs, d), rows, cols in (("gate", gate, ffn, hidden), ("up", up, ffn, hidden),
                                          ("down", down, hidden, ffn)):
            ptr += [_flat(qs, (E, rows, cols // 32, 16), torch.uint8, dev, f"MoeQ4_0: {what} quants"),
                    _flat(d, (E, rows, cols // 32), torch.float16, dev, f"MoeQ4_0: {what} scales")]
        self._keep = (router, bias, gate, up, down)
        self._dev, self._hidden, self._k = dev, hidden, int(top_k)
        self._desc = MoeDesc(E, int(top_k), hidden, ffn, ("sigmoid", "softmax").index(score), int(bool(renorm)),
                             float(scale), *ptr)
        self._ref = ctypes.addressof(self._desc)
        self.max_tokens = int(max_tokens)
        n = self.work_bytes()
        if dev < 0:
            raise ValueError("MoeQ4_0: tensors must live in device memory")
        self._work = torch.empty(n, dtype=torch.uint8, device=router.device)
        self._streams = {torch.cuda.current_stream(dev).cuda_stream}     # those that the workspace's memory is known to

    def work_bytes(self) -> int:
        """Bytes of workspace for max_tokens tokens."""
        n = int(load().lk_moe_work_bytes(self._ref, self.max_tokens))
        if n == 0:
            raise LkError(load().lk_last_error().decode(errors="replace"))
        return n

    def _tell(self, stream) -> None:
        """Tells the allocator of a stream that uses the layer's workspace, so that a layer dropped
        while the stream has work left does not give the memory away."""
        if stream is None and _raw_stream is not None and _raw_stream(self._dev) in self._streams:
            return
        s = _torch.cuda.current_stream(self._dev) if stream is None else stream
        if s.cuda_stream not in self._streams:
            self._work.record_stream(s)
            self._streams.add(s.cuda_stream)

    def __call__(self, x, out, res=None, ids=None, weights=None, work=None, stream=None) -> None:
        """out[t] = (res[t] +) the layer of x[t], rows [T][hidden] of fp32, fp16 or bf16
        (out may be x, res may be out); ids int32 and weights fp32 [T][top_k] where
        given.  Up to 8 tokens a row's last fp32 bits depend on the batch, from 9 on not."""
        ty = _type_of(x, "MoeQ4_0")
        if x.dim() != 2:
            raise ValueError("MoeQ4_0: x must be [tokens, hidden]")
        T, dev = x.shape[0], self._dev
        shape = (T, self._hidden)
        if T > self.max_tokens:
            raise ValueError(f"MoeQ4_0: {T} tokens, made for {self.max_tokens}")
        px, ldx = _rows2(x, shape, x.dtype, dev, "MoeQ4_0: x")
        po, ldo = _rows2(out, shape, x.dtype, dev, "MoeQ4_0: out")
        pr, ldr = _rows2(res, shape, x.dtype, dev, "MoeQ4_0: res")
        pi = None if ids is None else _flat(ids, (T, self._k), _torch.int32, dev, "MoeQ4_0: ids")
        pw = None if weights is None else _flat(weights, (T, self._k), _torch.float32, dev, "MoeQ4_0: weights")
        if work is None:
            work = self._work
        elif work.dtype is not _torch.uint8 or work.get_device() != dev or not work.is_contiguous():
            raise ValueError("MoeQ4_0: work must be contiguous uint8 on the layer's device")
        rc = _on(dev, stream, load().lk_moe_q4_0, self._ref, ty, px, ldx, T, pr, ldr, po, ldo, pi, pw,
                 work.data_ptr(), work.numel())
        if rc:
            _check(rc, "lk_moe_q4_0")
        if work is self._work:
            self._tell(stream)


# ---- many sequences over a paged cache ---------------------------------------------
ROPE_HALVES, ROPE_PAIRS = 0, 1


class Pages(ctypes.Structure):
    """lk_pages (include/lk_attn.h)."""
    _fields_ = [(n, ctypes.c_int) for n in ("type", "n_heads", "n_kv_heads", "head_dim", "page", "n_pages")] + \
        [("k", ctypes.c_void_p), ("v", ctypes.c_void_p)]


class Step(ctypes.Structure):
    """lk_step (include/lk_attn.h)."""
    _fields_ = [("n_seqs", ctypes.c_int), ("rows", ctypes.c_int)] + \
        [(n, ctypes.c_void_p) for n in ("first", "lens", "table")] + [("ldt", ctypes.c_int), ("width", ctypes.c_int)] + \
        [("pos", ctypes.c_void_p), ("mask", ctypes.c_void_p), ("max_new", ctypes.c_int)]


class PagedStep:
    """A step's tables (lk_step), shared by all layers: first int32 [n_seqs + 1], lens int32
    [n_seqs], table int32 [n_seqs][pages], `rows` rows of new tokens; pos int32 [rows] and
    mask int64 [rows] (64 bits a row) where given; max_new, the largest number of new tokens a
    sequence has, chooses a kernel (0: by rows a sequence).  The tables are read on the device during each call, so a
    captured call goes on with what they hold when it is replayed.
    Keeps the tables and the attention's workspace, made at its first use (or `work`, uint8 of
    PagedCache.work_bytes()): attention calls on a step must be ordered (one stream, or
    events); calls that may overlap, captured graphs among them, take steps of their own.  A step
    may be dropped while streams still work on it as far as a workspace of its own goes; a captured
    graph needs its steps kept."""

    def __init__(self, first, lens, table, rows: int, pos=None, mask=None, max_new: int = 0, work=None):
        import torch
        if lens.dim() != 1 or table.dim() != 2:
            raise ValueError("PagedStep: lens must be [sequences], table [sequences, pages]")
        B, dev, i32 = lens.shape[0], lens.get_device(), torch.int32
        if dev < 0:
            raise ValueError("PagedStep: tensors must live in device memory")
        pt, ldt = _rows2(table, (B, table.shape[1]), i32, dev, "PagedStep: table")
        self._desc = Step(B, int(rows), _flat(first, (B + 1,), i32, dev, "PagedStep: first"),
                          _flat(lens, (B,), i32, dev, "PagedStep: lens"), pt, ldt, table.shape[1],
                          None if pos is None else _flat(pos, (rows,), i32, dev, "PagedStep: pos"),
                          None if mask is None else _flat(mask, (rows,), torch.int64, dev, "PagedStep: mask"), int(max_new))
        if work is not None and (work.dtype is not torch.uint8 or work.get_device() != dev or not work.is_contiguous()):
            raise ValueError("PagedStep: work must be contiguous uint8 on the tables' device")
        self._ref = ctypes.addressof(self._desc)
        self._keep = (first, lens, table, pos, mask)
        self._dev, self.n_seqs, self.rows, self.max_new = dev, B, int(rows), int(max_new)
        self._most = self.max_new or (-(-self.rows // B) if B else 0)       # what lk_paged_attn takes for an unknown one
        self._work, self._own, self._streams, self._old = work, False, set(), []

    def _workspace(self, n: int, stream):
        """The workspace, of at least n bytes where it is the step's own; made on the stream of the call,
        whose turn on the memory is then the next one."""
        if self._work is None or (self._own and self._work.numel() < n):
            if getattr(stream, "device_index", self._dev) != self._dev:
                raise ValueError("lk_attn: the stream is one of another device than the tensors'")
            with _torch.cuda.device(self._dev), _torch.cuda.stream(stream):       # None: the current stream
                self._old.append(self._work)             # a captured call may still have it
                self._work = _torch.empty(n, dtype=_torch.uint8, device=self._keep[1].device)
                self._own = True
                self._streams = {_torch.cuda.current_stream(self._dev).cuda_stream}
        return self._work

    def _tell(self, stream) -> None:
        """Tells the allocator of a stream that uses the step's own workspace, so that a step dropped while
        the stream has work left does not give the memory away."""
        if stream is None and _raw_stream is not None and _raw_stream(self._dev) in self._streams:
            return
        s = _torch.cuda.current_stream(self._dev) if stream is None else stream
        if s.cuda_stream not in self._streams:
            self._work.record_stream(s)
            self._streams.add(s.cuda_stream)


class PagedCache:
    """A layer's paged KV cache: pools k and v, fp16 or bf16 [pages][positions a page][kv heads]
    [head_dim], read by n_heads query heads.  Rows are fp32 or fp16 with fp16 pools, bf16 with
    bf16 pools."""

    def __init__(self, k, v, n_heads: int):
        ty = _type_of(k, "PagedCache")
        if k.dim() != 4:
            raise ValueError("PagedCache: pools must be [pages, positions, kv heads, head_dim]")
        n, page, hkv, d = k.shape
        dev = k.get_device()
        if dev < 0:
            raise ValueError("PagedCache: tensors must live in device memory")
        self._desc = Pages(ty, int(n_heads), hkv, d, page, n, _flat(k, k.shape, k.dtype, dev, "PagedCache: k"),
                           _flat(v, k.shape, k.dtype, dev, "PagedCache: v"))
        self._ref = ctypes.addressof(self._desc)
        self.k, self.v = k, v
        self._dev, self._hq, self._hkv, self._d = dev, int(n_heads) * d, hkv * d, d
        self._scale, self._need = d ** -0.5, {}

    def work_bytes(self, dtype, max_new: int = 0) -> int:
        """Bytes of attention workspace for rows of a dtype."""
        n = self._need.get((dtype, max_new))
        if n is None:
            ty = _types.get(dtype)
            if ty is None:
                raise ValueError(f"PagedCache: fp32, fp16 or bf16 rows, not {dtype}")
            n = int(load().lk_paged_attn_work_bytes(self._ref, ty, int(max_new)))
            if n == 0:
                raise LkError(load().lk_last_error().decode(errors="replace"))
            self._need[(dtype, max_new)] = n
        return n

    def append(self, step, k, v, q=None, q_out=None, qn=None, kn=None, freq=None, eps: float = 1e-5, pairs: bool = False,
               stream=None) -> None:
        """k and v rows [rows][kv heads * head_dim] to their slots, k normed (weights kn fp32
        [head_dim], or None: not) and rotated (freq fp32 [pairs of values], or None: not; `pairs`:
        neighbouring values instead of halves); q [rows][heads * head_dim] the same with qn into
        q_out (which may be q) (lk_paged_append).  Rows may be parts of wider ones."""
        ty = _type_of(k, "PagedCache.append")
        rows, dev, dt = step.rows, self._dev, k.dtype
        pk, ldk = _rows2(k, (rows, self._hkv), dt, dev, "PagedCache.append: k")
        pv, ldv = _rows2(v, (rows, self._hkv), dt, dev, "PagedCache.append: v")
        pq, ldq = _rows2(q, (rows, self._hq), dt, dev, "PagedCache.append: q")
        po, ldo = _rows2(q_out, (rows, self._hq), dt, dev, "PagedCache.append: q_out")
        f32 = _torch.float32
        pqn = None if qn is None else _flat(qn, (self._d,), f32, dev, "PagedCache.append: qn")
        pkn = None if kn is None else _flat(kn, (self._d,), f32, dev, "PagedCache.append: kn")
        rot, pf = 0, None
        if freq is not None:
            rot, pf = 2 * freq.numel(), _flat(freq, (freq.numel(),), f32, dev, "PagedCache.append: freq")
        if step._dev != dev:
            raise ValueError("PagedCache: the step is on another device")
        rc = _on(dev, stream, (_lib or load()).lk_paged_append, self._ref, step._ref, ty, pq, ldq, pk, ldk, pv, ldv, pqn, pkn, eps,
                 pf, rot, ROPE_PAIRS if pairs else ROPE_HALVES, po, ldo)
        if rc:
            _check(rc, "lk_paged_append")

    def attend(self, step, q, out, scale: Optional[float] = None, cap: float = 0.0, slopes=None, stream=None) -> None:
        """out = attention of the step's rows q [rows][heads * head_dim] over their sequences' pages
        and new tokens, which may be written over q (lk_paged_attn); scale 1/sqrt(head_dim) unless given, cap > 0: scores capped
        by cap * tanh(x / cap), slopes fp32 [heads]: a bias of slope times distance."""
        ty = _type_of(q, "PagedCache.attend")
        shape, dev, dt = (step.rows, self._hq), self._dev, q.dtype
        pq, ldq = _rows2(q, shape, dt, dev, "PagedCache.attend: q")
        po, ldo = _rows2(out, shape, dt, dev, "PagedCache.attend: out")
        ps = None if slopes is None else _flat(slopes, (self._hq // self._d,), _torch.float32, dev, "PagedCache.attend: slopes")
        if step._dev != dev:
            raise ValueError("PagedCache: the step is on another device")
        work = step._workspace(self.work_bytes(dt, step._most), stream)
        rc = _on(dev, stream, (_lib or load()).lk_paged_attn, self._ref, step._ref, ty, pq, ldq,
                 self._scale if scale is None else scale, cap, ps, po, ldo, work.data_ptr(), work.numel())
        if rc:
            _check(rc, "lk_paged_attn")
        if step._own:
            step._tell(stream)

    def commit(self, step, path, count, new_lens, stream=None) -> None:
        """The accepted tokens of each sequence (places path int32 [sequences][most], strictly
        increasing, count int32 [sequences] of them; path None: the first count) become its next
        positions; new_lens int32 [sequences] (which may be the step's lens) (lk_paged_commit)."""
        i32, dev, B = _torch.int32, self._dev, step.n_seqs
        pp, ldp = None, 0
        if path is not None:
            ldp = path.shape[-1]
            pp = _flat(path, (B, ldp), i32, dev, "PagedCache.commit: path")
        if step._dev != dev:
            raise ValueError("PagedCache: the step is on another device")
        rc = _on(dev, stream, (_lib or load()).lk_paged_commit, self._ref, step._ref, pp, ldp,
                 _flat(count, (B,), i32, dev, "PagedCache.commit: count"),
                 _flat(new_lens, (B,), i32, dev, "PagedCache.commit: new_lens"))
        if rc:
            _check(rc, "lk_paged_commit")


class PrefillCtx:
    """lk_pf_ctx: the prefill chunk driver's state (int8 K copies, k8_valid)."""

    def __init__(self, n_layers, max_chunk, max_seq, attn8=True, ksmooth=False, near=1024, sink=1):
        h = ctypes.c_void_p()
        _check(load().lk_pf_ctx_create(int(n_layers), int(max_chunk), int(max_seq), int(bool(attn8)),
                                       int(bool(ksmooth)), int(near), int(sink), ctypes.byref(h)),
               "lk_pf_ctx_create")
        self._h = h

    def chunk_attn(self, layer, Y, qn, kn, m, pos0, kc, vc, o, aqs=None, asc=None, stream=None) -> None:
        _check(load().lk_pf_chunk_attn(self._h, int(layer), _ptr(Y), _ptr(qn), _ptr(kn), int(m), int(pos0),
                                       _ptr(kc), _ptr(vc), _ptr(o), _ptr(aqs), _ptr(asc), _stream(stream)),
               "lk_pf_chunk_attn")

    def chunk_done(self, pos_end) -> None:
        _check(load().lk_pf_chunk_done(self._h, int(pos_end)), "lk_pf_chunk_done")

    def buffers(self, layer) -> dict:
        qh, k8, ksc, cm = (ctypes.c_void_p() for _ in range(4))
        ks, kv = ctypes.c_int(), ctypes.c_int()
        _check(load().lk_pf_ctx_buffers(self._h, int(layer), ctypes.byref(qh), ctypes.byref(k8),
                                        ctypes.byref(ksc), ctypes.byref(cm), ctypes.byref(ks),
                                        ctypes.byref(kv)), "lk_pf_ctx_buffers")
        return {"qh": qh.value, "k8": k8.value, "ksc": ksc.value, "cm": cm.value,
                "kstride": ks.value, "k8_valid": kv.value}

    def close(self) -> None:
        if getattr(self, "_h", None):
            load().lk_pf_ctx_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
