"""ctypes binding of libkestrel_cuda.so (include/kestrel_cuda.h).

The Python mirror of the calls Kestrel's engine makes on its MoE path:
`Context.moe_ffn` is Transformer::moe_ffn (crates/kestrel-engine/src/
transformer.rs:513-589), `Context.matmul` is quant::matmul (quant.rs:229-339),
`Context.upload_experts` is ExpertStore::preload_all into HBM (crates/
kestrel-memory/src/expert.rs:620-641). The paged key-value cache and its attention
(`Context.kv_*`, `Context.attn_*`) are additions for servers. Failures raise `KestrelCudaError`
carrying the library's status code and message (the analogue of
EngineError, transformer.rs:15-27); there is no CPU fallback: if the CUDA
library is missing or fails to load, importing this module raises.
"""
from __future__ import annotations

import ctypes
import os

import numpy as np

from . import ggml as G

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libkestrel_cuda.so")

STATUS = {0: "OK", 1: "ERR_ARG", 2: "ERR_SHAPE", 3: "ERR_TYPE", 4: "ERR_CUDA", 5: "ERR_NCCL",
          6: "ERR_TIMEOUT", 7: "ERR_STATE", 8: "ERR_OOM"}

# Every symbol include/kestrel_cuda.h declares, with its ctypes signature.
P, I, I64, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
SIGNATURES = {
    "kc_init": (I, [I, ctypes.POINTER(P)]),
    "kc_free": (None, [P]),
    "kc_last_error": (ctypes.c_char_p, [P]),
    "kc_set_stream": (I, [P, P]),
    "kc_reserve": (I, [P, I]),
    "kc_sync": (I, [P]),
    "kc_device_bytes": (I64, [P]),
    "kc_upload_experts": (I, [P, I, I, I, I, I, P, I, P, I, P, I]),
    "kc_upload_experts_range": (I, [P, I, I, I, I, I, I, I, P, I, P, I, P, I]),
    "kc_upload_router": (I, [P, I, P, I, I, I, I, F, I]),
    "kc_upload_dense": (I, [P, I, I, P, I64, I64, I]),
    "kc_moe_ffn": (I, [P, I, P, I, P, I, I, I, F, P, P, P]),
    "kc_moe_ffn_dev": (I, [P, I, P, I, P, P, P]),
    "kc_matmul": (I, [P, I, P, I, P]),
    "kc_matmul_dev": (I, [P, I, P, I, P]),
    "kc_q8k_quantize_dev": (I, [P, P, I64, I64, P, P, P]),
    "kc_q8_quantize_dev": (I, [P, P, I64, I64, P, P, P]),
    "kc_route_dev": (I, [P, P, I, I, I, I, F, P, P]),
    "kc_router_logits_dev": (I, [P, P, I, I, P, I, P]),
    "kc_block_sums_dev": (I, [P, I, P, I64, I64, P, P, I, P]),
    "kc_quantize_dev": (I, [P, I, P, I64, I64, P]),
    "kc_profile_enable": (I, [P, I]),
    "kc_profile_read": (I, [P, P, P, I]),
    "kc_kernel_launches": (I64, []),
    "kc_route_noalloc": (I, [P, I, I, P, I, I, I, F, P, P, P]),
    "kc_upload_shared_expert": (I, [P, I, I, I, I, P, I, P, I, P, P, I]),
    "kc_ep_unique_id": (I, [ctypes.c_char_p]),
    "kc_ep_init": (I, [P, I, I, ctypes.c_char_p]),
    "kc_ep_reserve": (I, [P, I]),
    "kc_set_option": (I, [P, I, I]),
    "kc_model_init": (I, [P, I, I, I, I, I, I, I, I, F, F, I]),
    "kc_model_tensor": (I, [P, I, I, I, P, I64, I64, I]),
    "kc_model_forward": (I, [P, P, I, P, P]),
    "kc_model_generate": (I, [P, P, I, I, P]),
    "kc_model_generate_batch": (I, [P, I, P, P, I, P]),
    "kc_model_set_sequences": (I, [P, I]),
    "kc_model_prefill_seq": (I, [P, I, P, I, P]),
    "kc_model_decode_seqs": (I, [P, I, I, P]),
    "kc_model_truncate": (I, [P, I]),
    "kc_model_cached": (I, [P]),
    "kc_load_gguf": (I, [P, ctypes.c_char_p, I, ctypes.c_char_p, I64]),
    "kc_gguf_inspect": (I, [ctypes.c_char_p, ctypes.c_char_p, I64]),
    "kc_upload_experts_streamed": (I, [P, I, I, I, I, I, P, I, P, I, P, I]),
    "kc_expert_cache_reserve": (I, [P, I, I, I, I]),
    "kc_expert_prefetch": (I, [P, I, P, I]),
    "kc_expert_cache_stats": (I, [P, P, I]),
    "kc_expert_cache_decay": (I, [P]),
    "kc_kv_cache": (I, [P, I, I, I, I, I, I, I, I, I, P, P, P, P, P]),
    "kc_kv_drop": (I, [P, I]),
    "kc_kv_fork_dev": (I, [P, I, P, P, I]),
    "kc_kv_extend_dev": (I, [P, I, P, P, I]),
    "kc_kv_write_dev": (I, [P, I, I, P, P, I, I, I, P, P, I64, I64]),
    "kc_kv_free_dev": (I, [P, I, P, P, I]),
    "kc_kv_compact_dev": (I, [P, I, P]),
    "kc_kv_copy_pages_dev": (I, [P, I, P, P, I]),
    "kc_attn_decode_dev": (I, [P, I, I, P, I, I, I, P, I64, F, I, I, P, I64]),
    "kc_attn_prompt_dev": (I, [P, I, I, P, P, I, I, I, I, P, I64, F, I, I, P, I64]),
}

# Options (kc_set_option) and whole-model tensor kinds (kc_model_tensor).
OPT_F32_PREFILL = 1
OPT_LOOKAHEAD = 2
# Expert-cache policies (kc_expert_cache_reserve) and counters (kc_expert_cache_stats).
EXPERT_POLICY_LFRU, EXPERT_POLICY_LRU = 0, 1
XS_COUNTERS = ["capacity", "cached", "requests", "hits", "late", "misses", "scratch_loads", "bytes_read",
               "prefetch_issued", "prefetch_used", "prefetch_wasted", "evictions", "lookahead_predicted",
               "lookahead_correct", "reads", "forced", "scratch", "spec", "spec_pauses"]
ARCH_LLAMA, ARCH_QWEN2, ARCH_QWEN3 = 0, 1, 2
(T_ATTN_NORM, T_ATTN_Q, T_ATTN_K, T_ATTN_V, T_ATTN_OUT, T_ATTN_Q_BIAS, T_ATTN_K_BIAS, T_ATTN_V_BIAS,
 T_ATTN_Q_NORM, T_ATTN_K_NORM, T_FFN_NORM, T_FFN_GATE, T_FFN_UP, T_FFN_DOWN) = range(14)
T_TOKEN_EMBD, T_OUTPUT_NORM, T_OUTPUT = 0, 1, 2


class KestrelCudaError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"{STATUS.get(code, code)}: {msg}")
        self.code = code


def load_library(path: str = LIB_PATH) -> ctypes.CDLL:
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: build it with `python -m kestrel_b200.build` "
                          "(there is no CPU fallback for the CUDA path)")
    lib = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return lib


_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        _lib = load_library()
    return _lib


def _ptr(a):
    """Address of a numpy array or a torch tensor (host or device). For a
    writable numpy array the address comes through the buffer protocol
    (several times cheaper than ndarray.ctypes, which builds a helper object
    per call: it matters on the per-call path); read-only, empty or
    non-contiguous arrays take ndarray.ctypes."""
    if a is None:
        return None
    if isinstance(a, np.ndarray):
        try:
            return ctypes.addressof(ctypes.c_char.from_buffer(a))
        except (TypeError, ValueError, BufferError):
            return a.ctypes.data
    return a.data_ptr()


def _is_dev(a) -> bool:
    return not isinstance(a, np.ndarray) and getattr(a, "is_cuda", False)


def _host_u8(a):
    return np.ascontiguousarray(a, dtype=np.uint8).reshape(-1) if isinstance(a, np.ndarray) else a


# ggml ids of the element types the paged cache takes: by torch's name, and by
# the dtype objects seen so far (these helpers are on the per-call path).
_FLOAT_NAMES = {"torch.float32": G.F32, "torch.float16": G.F16, "torch.bfloat16": G.BF16}
_FLOAT_TYPES = {}


def _float_type(name: str, a) -> int:
    t = _FLOAT_TYPES.get(a.dtype)
    if t is None:
        t = _FLOAT_NAMES.get(str(a.dtype))
        if t is None:
            raise ValueError(f"{name} must be float32, float16 or bfloat16, not {a.dtype}")
        _FLOAT_TYPES[a.dtype] = t
    return t


_INT32 = set()  # torch.int32, once seen


def _dev_ints(name: str, a, size: int | None = None):
    """A contiguous int32 CUDA tensor of `size` values (None: any)."""
    if a is None:
        return None
    if not _is_dev(a) or not (a.dtype in _INT32 or str(a.dtype) == "torch.int32") or not a.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 CUDA tensor")
    _INT32.add(a.dtype)
    if size is not None and a.numel() != size:
        raise ValueError(f"{name} holds {a.numel()} values, {size} needed")
    return a.data_ptr()


def _dev_rows(name: str, a, heads: int | None = None, head_dim: int | None = None):
    """Row stride (elements) of a CUDA tensor [rows, heads, head_dim] whose
    heads are contiguous within a row."""
    shape = a.shape
    if not _is_dev(a) or len(shape) != 3 or (heads is not None and shape[1] != heads) or \
            (head_dim is not None and shape[2] != head_dim):
        raise ValueError(f"{name} must be a CUDA tensor [rows, heads, head_dim]")
    rows, nh, hd = shape
    stride = a.stride()
    if (hd > 1 and stride[2] != 1) or (nh > 1 and stride[1] != hd):
        raise ValueError(f"the heads of a row of {name} must be contiguous")
    return stride[0] if rows > 1 else nh * hd


class Context:
    """One GPU's backend context (kc_ctx)."""

    def __init__(self, device: int = 0):
        h = ctypes.c_void_p()
        rc = lib().kc_init(device, ctypes.byref(h))
        if rc != 0:
            raise KestrelCudaError(rc, lib().kc_last_error(None).decode())
        self.h = h
        self.device = device
        self._k = {}           # layer -> top-k of its uploaded router
        self._dense_rows = {}  # tensor id -> rows
        self._kv = {}          # paged cache id -> its tensors (kept alive while registered)
        self._kv_dims = {}     # and (sequences, key-value heads, head size)

    def close(self):
        if getattr(self, "h", None):
            lib().kc_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc: int):
        if rc != 0:
            raise KestrelCudaError(rc, lib().kc_last_error(self.h).decode())

    # ---- set-up --------------------------------------------------------
    def reserve(self, max_tokens: int):
        self._check(lib().kc_reserve(self.h, max_tokens))

    def set_stream(self, stream_ptr: int | None):
        self._check(lib().kc_set_stream(self.h, stream_ptr))

    def sync(self):
        self._check(lib().kc_sync(self.h))

    def device_bytes(self) -> int:
        return int(lib().kc_device_bytes(self.h))

    def upload_experts(self, layer: int, n_expert: int, d: int, ff: int, t_gate: int, gate, t_up: int, up,
                       t_down: int, down, first_expert: int = 0, n_local: int | None = None):
        """Stacked GGUF expert tensors (numpy host bytes or torch CUDA uint8)."""
        n_local = n_expert if n_local is None else n_local
        gate, up, down = _host_u8(gate), _host_u8(up), _host_u8(down)
        dev = _is_dev(gate)
        for t, a, rows, cols in ((t_gate, gate, ff, d), (t_up, up, ff, d), (t_down, down, d, ff)):
            want = n_local * rows * G.bytes_for(t, cols)
            n = a.size if isinstance(a, np.ndarray) else a.numel() * a.element_size()
            if n < want:
                raise ValueError(f"expert tensor holds {n} bytes, {want} needed")
        self._check(lib().kc_upload_experts_range(self.h, layer, n_expert, first_expert, n_local, d, ff, t_gate,
                                                  _ptr(gate), t_up, _ptr(up), t_down, _ptr(down), int(dev)))

    def upload_experts_streamed(self, layer: int, n_expert: int, d: int, ff: int, t_gate: int, gate, t_up: int,
                                up, t_down: int, down):
        """Like upload_experts, but the experts stay in pinned host memory and
        each call copies the ones it routes to into HBM slots."""
        gate, up, down = _host_u8(gate), _host_u8(up), _host_u8(down)
        dev = _is_dev(gate)
        for t, a, rows, cols in ((t_gate, gate, ff, d), (t_up, up, ff, d), (t_down, down, d, ff)):
            want = n_expert * rows * G.bytes_for(t, cols)
            n = a.size if isinstance(a, np.ndarray) else a.numel() * a.element_size()
            if n < want:
                raise ValueError(f"expert tensor holds {n} bytes, {want} needed")
        self._check(lib().kc_upload_experts_streamed(self.h, layer, n_expert, d, ff, t_gate, _ptr(gate), t_up,
                                                     _ptr(up), t_down, _ptr(down), int(dev)))

    def expert_cache_reserve(self, capacity: int, scratch: int = 0, policy: int = EXPERT_POLICY_LFRU,
                             spec: int | None = None):
        """spec: speculative slots (default max(1, scratch), as ExpertStore::new sets)."""
        spec = max(1, scratch) if spec is None else spec
        self._check(lib().kc_expert_cache_reserve(self.h, capacity, scratch, spec, policy))

    def expert_prefetch(self, layer: int, experts):
        ids = np.ascontiguousarray(np.asarray(experts, dtype=np.int32))
        self._check(lib().kc_expert_prefetch(self.h, layer, ids.ctypes.data, ids.size))

    def expert_cache_stats(self) -> dict:
        out = np.zeros(len(XS_COUNTERS), np.uint64)
        self._check(lib().kc_expert_cache_stats(self.h, out.ctypes.data, out.size))
        return {k: int(v) for k, v in zip(XS_COUNTERS, out)}

    def expert_cache_decay(self):
        self._check(lib().kc_expert_cache_decay(self.h))

    def upload_router(self, layer: int, router_w, k: int, norm_topk: bool = True, weights_scale: float = 0.0):
        rw = router_w if _is_dev(router_w) else np.ascontiguousarray(router_w, dtype=np.float32)
        E, d = rw.shape
        self._check(lib().kc_upload_router(self.h, layer, _ptr(rw), E, d, k, int(norm_topk), weights_scale,
                                           int(_is_dev(rw))))
        self._k[layer] = k

    def upload_shared_expert(self, layer: int, ff: int, d: int, t_gate: int, gate, t_up: int, up, t_down: int,
                             down, gate_inp=None):
        """qwen2moe shared expert of `layer` (host numpy GGUF bytes or torch CUDA
        uint8); gate_inp: optional F32 [d] gate vector."""
        gate, up, down = _host_u8(gate), _host_u8(up), _host_u8(down)
        dev = _is_dev(gate)
        gi = None if gate_inp is None else (gate_inp if _is_dev(gate_inp) else
                                            np.ascontiguousarray(gate_inp, dtype=np.float32))
        self._check(lib().kc_upload_shared_expert(self.h, layer, ff, d, t_gate, _ptr(gate), t_up, _ptr(up), t_down,
                                                  _ptr(down), _ptr(gi), int(dev)))

    def upload_dense(self, tensor_id: int, t: int, w, rows: int, cols: int):
        w = _host_u8(w) if t != G.F32 or not isinstance(w, np.ndarray) else \
            np.ascontiguousarray(w, dtype=np.float32)
        self._check(lib().kc_upload_dense(self.h, tensor_id, t, _ptr(w), rows, cols, int(_is_dev(w))))
        self._dense_rows[tensor_id] = rows

    # ---- hot path (host buffers) -------------------------------------------
    def moe_ffn(self, layer: int, h, router_w=None, k: int = 0, norm_topk: bool = True,
                weights_scale: float = 0.0, out=None, topk: bool = True):
        """Transformer::moe_ffn on host f32 h [n, d] -> (out, topk ids, topk w).
        `out`: optional caller buffer (e.g. pinned) for the result; with
        topk=False the ids and weights are not copied back (returned as None)."""
        h = np.ascontiguousarray(h, dtype=np.float32)
        n, d = h.shape
        rw = None if router_w is None else np.ascontiguousarray(router_w, dtype=np.float32)
        E = 0 if rw is None else rw.shape[0]
        kk = k if rw is not None else self._layer_k(layer)
        if out is None:
            out = np.empty((n, d), np.float32)
        elif out.dtype != np.float32 or out.shape != (n, d) or not out.flags.c_contiguous:
            raise ValueError("out must be a C-contiguous float32 [n, d] array")
        ids = np.empty((n, kk), np.int32) if topk else None
        w = np.empty((n, kk), np.float32) if topk else None
        self._check(lib().kc_moe_ffn(self.h, layer, _ptr(h), n, _ptr(rw), E, k, int(norm_topk), weights_scale,
                                     _ptr(out), _ptr(ids), _ptr(w)))
        return out, ids, w

    def _layer_k(self, layer):
        if layer not in self._k:
            raise ValueError("router not uploaded through this Context; pass router_w and k")
        return self._k[layer]

    def matmul(self, tensor_id: int, x) -> np.ndarray:
        x = np.ascontiguousarray(x, dtype=np.float32)
        rows = self._dense_rows[tensor_id]
        out = np.empty((x.shape[0], rows), np.float32)
        self._check(lib().kc_matmul(self.h, tensor_id, _ptr(x), x.shape[0], _ptr(out)))
        return out

    # ---- device buffers (torch CUDA tensors) ---------------------------------
    def moe_ffn_dev(self, layer: int, h, out, ids=None, w=None, n_tok: int | None = None):
        n = h.shape[0] if n_tok is None else n_tok
        self._check(lib().kc_moe_ffn_dev(self.h, layer, _ptr(h), n, _ptr(out), _ptr(ids), _ptr(w)))

    def matmul_dev(self, tensor_id: int, x, out, n: int | None = None):
        self._check(lib().kc_matmul_dev(self.h, tensor_id, _ptr(x), x.shape[0] if n is None else n, _ptr(out)))

    def q8k_quantize_dev(self, x, q, d, bsums):
        self._check(lib().kc_q8k_quantize_dev(self.h, _ptr(x), x.shape[0], x.shape[1], _ptr(q), _ptr(d),
                                              _ptr(bsums)))

    def q8_quantize_dev(self, x, q, d, s16):
        self._check(lib().kc_q8_quantize_dev(self.h, _ptr(x), x.shape[0], x.shape[1], _ptr(q), _ptr(d),
                                             _ptr(s16)))

    def route_dev(self, logits, k: int, ids, w, norm_topk: bool = True, weights_scale: float = 0.0):
        n, E = logits.shape
        self._check(lib().kc_route_dev(self.h, _ptr(logits), n, E, k, int(norm_topk), weights_scale, _ptr(ids),
                                       _ptr(w)))

    def router_logits_dev(self, router_w, h, logits):
        E, d = router_w.shape
        self._check(lib().kc_router_logits_dev(self.h, _ptr(router_w), E, d, _ptr(h), h.shape[0], _ptr(logits)))

    def block_sums_dev(self, t: int, w, rows: int, cols: int, q, bsums, n_act: int, out):
        self._check(lib().kc_block_sums_dev(self.h, t, _ptr(w), rows, cols, _ptr(q), _ptr(bsums), n_act,
                                            _ptr(out)))

    def quantize_dev(self, t: int, x, out):
        rows, cols = x.shape
        self._check(lib().kc_quantize_dev(self.h, t, _ptr(x), rows, cols, _ptr(out)))

    STAGES = ["router_logits", "route", "dispatch", "quant_x", "gate_up_int8", "gate_up_f32", "quant_act",
              "down_int8", "down_f32", "combine", "expert_load"]

    def profile_enable(self, on: bool = True):
        self._check(lib().kc_profile_enable(self.h, int(on)))

    def profile_read(self) -> dict:
        """{stage: (total ms, calls)} accumulated since the previous read."""
        n = len(self.STAGES)
        ms = np.zeros(n, np.float64)
        calls = np.zeros(n, np.int64)
        self._check(lib().kc_profile_read(self.h, ms.ctypes.data, calls.ctypes.data, n))
        return {s: (float(ms[i]), int(calls[i])) for i, s in enumerate(self.STAGES)}

    def ep_init(self, rank: int, world: int, uid: bytes):
        self._check(lib().kc_ep_init(self.h, rank, world, uid))

    # ---- whole model (dense decode path) ---------------------------------------
    def set_option(self, option: int, value: int):
        self._check(lib().kc_set_option(self.h, option, int(value)))

    def model_init(self, n_layer: int, d: int, n_head: int, n_head_kv: int, head_dim: int, n_vocab: int,
                   n_ctx: int, rope_dim: int, rope_base: float, rms_eps: float, arch: int):
        self._n_vocab = n_vocab
        self._check(lib().kc_model_init(self.h, n_layer, d, n_head, n_head_kv, head_dim, n_vocab, n_ctx, rope_dim,
                                        rope_base, rms_eps, arch))

    def model_tensor(self, layer: int, kind: int, t: int, w, rows: int, cols: int):
        """A model tensor (layer -1) or a layer tensor; host numpy bytes / f32
        or a torch CUDA tensor."""
        if _is_dev(w):
            self._check(lib().kc_model_tensor(self.h, layer, kind, t, _ptr(w), rows, cols, 1))
            return
        a = np.ascontiguousarray(w, dtype=np.float32) if t == G.F32 else _host_u8(w)
        self._check(lib().kc_model_tensor(self.h, layer, kind, t, _ptr(a), rows, cols, 0))

    def model_forward(self, tokens):
        """Transformer::forward: logits of the last token (and its argmax)."""
        tk = np.ascontiguousarray(tokens, dtype=np.uint32)
        logits = np.empty(self._n_vocab, np.float32)
        nxt = np.zeros(1, np.uint32)
        self._check(lib().kc_model_forward(self.h, _ptr(tk), tk.size, _ptr(logits), _ptr(nxt)))
        return logits, int(nxt[0])

    def model_generate(self, prompt, n_gen: int):
        tk = np.ascontiguousarray(prompt, dtype=np.uint32)
        out = np.zeros(max(1, n_gen), np.uint32)
        self._check(lib().kc_model_generate(self.h, _ptr(tk), tk.size, n_gen, _ptr(out)))
        return [int(t) for t in out[:n_gen]]

    def model_generate_batch(self, prompts, n_gen: int):
        """kc_model_generate_batch: greedy decode of len(prompts) independent
        sequences in lockstep; returns one token list per sequence."""
        lens = np.array([len(p) for p in prompts], dtype=np.int32)
        flat = np.ascontiguousarray(np.concatenate([np.asarray(p, dtype=np.uint32) for p in prompts]))
        out = np.zeros((len(prompts), max(1, n_gen)), np.uint32)
        self._check(lib().kc_model_generate_batch(self.h, len(prompts), _ptr(flat), _ptr(lens), n_gen, _ptr(out)))
        return [[int(t) for t in row[:n_gen]] for row in out]

    def model_set_sequences(self, n_seq: int):
        self._check(lib().kc_model_set_sequences(self.h, n_seq))

    def model_prefill_seq(self, seq: int, prompt) -> int:
        """kc_model_prefill_seq: the prompt alone in sequence `seq`'s cache;
        returns its greedy next token (the sequence's pending token)."""
        tk = np.ascontiguousarray(prompt, dtype=np.uint32)
        nxt = np.zeros(1, np.uint32)
        self._check(lib().kc_model_prefill_seq(self.h, seq, _ptr(tk), tk.size, _ptr(nxt)))
        return int(nxt[0])

    def model_decode_seqs(self, n_seq: int, n_gen: int):
        out = np.zeros((n_seq, max(1, n_gen)), np.uint32)
        self._check(lib().kc_model_decode_seqs(self.h, n_seq, n_gen, _ptr(out)))
        return [[int(t) for t in row[:n_gen]] for row in out]

    def model_truncate(self, keep: int):
        self._check(lib().kc_model_truncate(self.h, keep))

    def model_cached(self) -> int:
        return int(lib().kc_model_cached(self.h))

    def load_gguf(self, path: str, n_ctx: int) -> dict:
        """kc_load_gguf: declare and upload a GGUF / KGUF model; returns the
        loader's summary (weight, KV-cache and free bytes)."""
        import json
        buf = ctypes.create_string_buffer(4096)
        rc = lib().kc_load_gguf(self.h, os.fsencode(path), n_ctx, buf, len(buf))
        info = json.loads(buf.value.decode()) if buf.value else {}
        self._check(rc)
        self._n_vocab = int(info.get("n_vocab", getattr(self, "_n_vocab", 0)))
        return info

    # ---- paged key-value cache (torch CUDA tensors) ------------------------------
    def kv_cache(self, cache: int, k, v, table, length, refs):
        """Register the caller's tensors as paged cache `cache`: k and v
        [n_layer, n_pages, n_kv, page, head_dim], table [n_seq, max_pages],
        length [n_seq] and refs [n_pages] int32 (an empty cache: -1, 0, 0).
        They stay the caller's; the calls below change them in stream order."""
        if not _is_dev(k) or not _is_dev(v) or k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype \
                or not k.is_contiguous() or not v.is_contiguous():
            raise ValueError("k and v must be contiguous CUDA tensors [n_layer, n_pages, n_kv, page, head_dim] of "
                             "one type")
        n_layer, n_pages, n_kv, page, hd = k.shape
        if table.dim() != 2:
            raise ValueError("table must be [n_seq, max_pages]")
        n_seq, max_pages = table.shape
        t = _dev_ints("table", table), _dev_ints("length", length, n_seq), _dev_ints("refs", refs, n_pages)
        self._check(lib().kc_kv_cache(self.h, cache, _float_type("k", k), n_layer, n_pages, page, n_kv, hd, n_seq,
                                      max_pages, k.data_ptr(), v.data_ptr(), *t))
        self._kv[cache] = (k, v, table, length, refs)
        self._kv_dims[cache] = (n_seq, n_kv, hd)

    def kv_drop(self, cache: int):
        self._check(lib().kc_kv_drop(self.h, cache))
        self._kv.pop(cache, None)
        self._kv_dims.pop(cache, None)

    def _kv_shape(self, cache: int):
        """(n_seq, n_kv, head_dim) of a registered cache."""
        dims = self._kv_dims.get(cache)
        if dims is None:
            raise ValueError(f"paged cache {cache} is not registered through this Context")
        return dims

    def kv_fork_dev(self, cache: int, src, dst):
        """Sequences dst (int32 CUDA tensor, empty ones) share the pages of src."""
        n = src.numel()
        self._check(lib().kc_kv_fork_dev(self.h, cache, _dev_ints("src", src), _dev_ints("dst", dst, n), n))

    def kv_extend_dev(self, cache: int, seqs, n_new):
        """n_new more positions for each of `seqs` (None: sequences 0, 1, ...)."""
        n = n_new.numel()
        self._check(lib().kc_kv_extend_dev(self.h, cache, _dev_ints("seqs", seqs, n), _dev_ints("n_new", n_new), n))

    def kv_write_dev(self, cache: int, layer: int, k, v, seqs=None, row_start=None):
        """Rows k, v [rows, n_kv, head_dim] become the last positions of their
        sequences: one row each, or rows row_start[i] .. row_start[i+1]-1."""
        _, n_kv, hd = self._kv_shape(cache)
        ks, vs = _dev_rows("k", k, n_kv, hd), _dev_rows("v", v, n_kv, hd)
        rows = k.shape[0]
        if v.shape[0] != rows or v.dtype != k.dtype:
            raise ValueError("k and v differ in rows or type")
        n = rows if row_start is None else row_start.numel() - 1
        self._check(lib().kc_kv_write_dev(self.h, cache, layer, _dev_ints("seqs", seqs, n),
                                          _dev_ints("row_start", row_start), n, rows, _float_type("k", k),
                                          k.data_ptr(), v.data_ptr(), ks, vs))

    def kv_free_dev(self, cache: int, seqs=None, keep=None):
        """Forget positions keep[i] and on (None: all) of each of `seqs` (None:
        every sequence, or the first len(keep))."""
        n = seqs.numel() if seqs is not None else keep.numel() if keep is not None else self._kv_shape(cache)[0]
        self._check(lib().kc_kv_free_dev(self.h, cache, _dev_ints("seqs", seqs), _dev_ints("keep", keep, n), n))

    def kv_compact_dev(self, cache: int, n_live=None):
        """Move the live pages to the front of the pool; n_live (int32 [1],
        optional) gets their number."""
        self._check(lib().kc_kv_compact_dev(self.h, cache, _dev_ints("n_live", n_live, 1)))

    def kv_copy_pages_dev(self, cache: int, src, dst):
        n = src.numel()
        self._check(lib().kc_kv_copy_pages_dev(self.h, cache, _dev_ints("src", src), _dev_ints("dst", dst, n), n))

    def _attn(self, cache, q, out):
        hd = self._kv_shape(cache)[2]
        qs, os_ = _dev_rows("q", q, None, hd), _dev_rows("out", out, None, hd)
        shape = q.shape
        if out.shape != shape or out.dtype != q.dtype:
            raise ValueError("out must have q's shape and type")
        return shape[0], shape[1], hd, qs, os_

    def attn_decode_dev(self, cache: int, layer: int, q, out, seqs=None, scale: float | None = None,
                        window: int = 0, sinks: int = 0):
        """Row i of q [n, n_head, head_dim] attends from the last position of
        sequence seqs[i]; scale None: head_dim ** -0.5."""
        n, nh, hd, qs, os_ = self._attn(cache, q, out)
        self._check(lib().kc_attn_decode_dev(self.h, cache, layer, _dev_ints("seqs", seqs, n), n, nh,
                                             _float_type("q", q), q.data_ptr(), qs,
                                             hd ** -0.5 if scale is None else scale, window, sinks, out.data_ptr(),
                                             os_))

    def attn_prompt_dev(self, cache: int, layer: int, q, row_start, out, seqs=None, scale: float | None = None,
                        window: int = 0, sinks: int = 0):
        """Rows row_start[i] .. row_start[i+1]-1 of q attend from the last
        positions of sequence seqs[i], causally."""
        rows, nh, hd, qs, os_ = self._attn(cache, q, out)
        n = row_start.numel() - 1
        self._check(lib().kc_attn_prompt_dev(self.h, cache, layer, _dev_ints("seqs", seqs, n),
                                             _dev_ints("row_start", row_start), n, rows, nh, _float_type("q", q),
                                             q.data_ptr(), qs, hd ** -0.5 if scale is None else scale, window, sinks,
                                             out.data_ptr(), os_))

    def ep_reserve(self, max_tokens: int):
        """Collective: map the peer exchange arenas for up to max_tokens tokens
        per rank and call (after uploading the layers)."""
        self._check(lib().kc_ep_reserve(self.h, max_tokens))


def gguf_inspect(path: str) -> dict:
    """kc_gguf_inspect: parse a GGUF / KGUF file (no GPU needed)."""
    import json
    cap = 1 << 22
    buf = ctypes.create_string_buffer(cap)
    rc = lib().kc_gguf_inspect(os.fsencode(path), buf, cap)
    if rc != 0:
        raise KestrelCudaError(rc, (lib().kc_last_error(None) or b"").decode())
    return json.loads(buf.value.decode())


def ep_unique_id() -> bytes:
    buf = ctypes.create_string_buffer(128)
    rc = lib().kc_ep_unique_id(buf)
    if rc != 0:
        raise KestrelCudaError(rc, "ncclGetUniqueId failed")
    return buf.raw


def kernel_launches() -> int:
    """CUDA kernels this library has launched in the process so far
    (kc_kernel_launches)."""
    return int(lib().kc_kernel_launches())
