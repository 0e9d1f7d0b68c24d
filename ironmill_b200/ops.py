"""Kernel-level entry points of the C ABI, called with torch CUDA tensors.

torch supplies device memory and streams only; every computation below is a call into
libironmill_cuda.so.  Names follow the reference's kernels
(crates/ironmill-inference/src/metal/shaders/**) and quantizer
(crates/mil-rs/src/ir/passes/affine_quantize.rs).
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from ._lib import IM_DTYPE_BF16, IM_DTYPE_F16, IM_DTYPE_F32, PagedKvStruct, check, lib, vp


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


class Device:
    """MetalDevice counterpart (crates/ironmill-metal-sys/src/device.rs:74-260)."""

    def __init__(self, ordinal: int = 0):
        self.handle = C.c_void_p()
        check(lib().im_cuda_device_open(C.c_int(ordinal), C.byref(self.handle)))
        self.ordinal = ordinal
        self.torch_device = torch.device("cuda", ordinal)
        self.select_bytes = {}  # scratch of beam_select, by sizes

    @property
    def name(self) -> str:
        buf = C.create_string_buffer(256)
        check(lib().im_cuda_device_name(self.handle, buf, C.c_size_t(256)))
        return buf.value.decode()

    @property
    def sm_count(self) -> int:
        return int(lib().im_cuda_device_sm_count(self.handle))

    def allocated_bytes(self) -> int:
        return int(lib().im_cuda_device_allocated_bytes(self.handle))

    def synchronize(self) -> None:
        check(lib().im_cuda_device_synchronize(self.handle))

    def close(self) -> None:
        if self.handle:
            lib().im_cuda_device_free(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Buffer:
    """MetalBuffer counterpart (crates/ironmill-metal-sys/src/buffer.rs:42-158)."""

    def __init__(self, dev: Device, nbytes: int, data: bytes | None = None):
        self.handle = C.c_void_p()
        if data is None:
            check(lib().im_cuda_buffer_alloc(dev.handle, C.c_size_t(nbytes), C.byref(self.handle)))
        else:
            check(lib().im_cuda_buffer_alloc_with_data(dev.handle, data, C.c_size_t(len(data)), C.byref(self.handle)))

    def __len__(self):
        return int(lib().im_cuda_buffer_length(self.handle))

    @property
    def ptr(self) -> int:
        return int(lib().im_cuda_buffer_ptr(self.handle) or 0)

    def write_bytes(self, data: bytes, offset: int = 0) -> None:
        check(lib().im_cuda_buffer_upload(self.handle, C.c_size_t(offset), data, C.c_size_t(len(data))))

    def read_bytes(self, nbytes: int, offset: int = 0) -> bytes:
        out = C.create_string_buffer(nbytes)
        check(lib().im_cuda_buffer_download(self.handle, C.c_size_t(offset), out, C.c_size_t(nbytes)))
        return out.raw

    def free(self):
        if self.handle:
            lib().im_cuda_buffer_free(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def quantize_affine(w: torch.Tensor, group_size: int, bit_width: int, awq: torch.Tensor | None = None):
    """GPU quantize + pack.  w fp16 [rows, K] -> (packed u8, scales f32 [rows,G], zps f32 [rows,G])."""
    assert w.is_cuda and w.dtype == torch.float16 and w.is_contiguous()
    rows = int(np.prod(w.shape[:-1])) if w.dim() > 1 else 1
    K = w.shape[-1] if w.dim() else 0
    G = -(-K // group_size) if K else 0
    total = rows * K
    nbytes = (total + 1) // 2 if bit_width == 4 else total
    packed = torch.empty(nbytes, dtype=torch.uint8, device=w.device)
    scales = torch.empty((rows, G), dtype=torch.float32, device=w.device)
    zps = torch.empty((rows, G), dtype=torch.float32, device=w.device)
    check(lib().im_cuda_quantize_affine(vp(w), vp(awq), C.c_size_t(rows), C.c_size_t(K), C.c_int(group_size),
                                        C.c_int(bit_width), vp(packed), vp(scales), vp(zps), _stream()))
    return packed, scales, zps


class AffineWeight:
    """GPU-resident affine-quantized weight (AffineQuantizedWeight,
    crates/ironmill-inference/src/metal/weights.rs:129-147)."""

    def __init__(self, dev: Device, qdata, scales, zeros, N: int, K: int, group_size: int, bit_width: int, awq=None):
        self.dev = dev
        self.N, self.K, self.group_size, self.bit_width = N, K, group_size, bit_width
        self.handle = C.c_void_p()
        if isinstance(qdata, torch.Tensor):
            assert qdata.is_cuda and scales.is_cuda and zeros.is_cuda
            pd = IM_DTYPE_F32 if scales.dtype == torch.float32 else IM_DTYPE_F16
            assert scales.dtype == zeros.dtype and scales.is_contiguous() and zeros.is_contiguous()
            check(lib().im_cuda_affine_weight_create_dev(dev.handle, vp(qdata), vp(scales), vp(zeros), C.c_int(pd),
                                                         vp(awq), C.c_int(N), C.c_int(K), C.c_int(group_size),
                                                         C.c_int(bit_width), _stream(), C.byref(self.handle)))
            torch.cuda.current_stream().synchronize()
        else:
            qdata = np.ascontiguousarray(qdata)
            scales = np.ascontiguousarray(scales)
            zeros = np.ascontiguousarray(zeros)
            assert scales.dtype == zeros.dtype and scales.dtype in (np.float32, np.float16)
            pd = IM_DTYPE_F32 if scales.dtype == np.float32 else IM_DTYPE_F16
            if awq is not None:
                awq = np.ascontiguousarray(awq)
                assert awq.dtype == np.float16
            check(lib().im_cuda_affine_weight_create(dev.handle, vp(qdata), vp(scales), vp(zeros), C.c_int(pd), vp(awq),
                                                     C.c_int(N), C.c_int(K), C.c_int(group_size), C.c_int(bit_width),
                                                     C.byref(self.handle)))

    def nbytes(self) -> int:
        return int(lib().im_cuda_affine_weight_bytes(self.handle))

    def dequant(self) -> torch.Tensor:
        out = torch.empty((self.N, self.K), dtype=torch.float16, device=f"cuda:{self.dev.ordinal}")
        check(lib().im_cuda_affine_weight_dequant(self.handle, vp(out), _stream()))
        return out

    def free(self):
        if self.handle:
            lib().im_cuda_affine_weight_free(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def _rows(x: torch.Tensor, K: int) -> int:
    assert x.is_cuda and x.dtype == torch.float16 and x.is_contiguous()
    assert x.shape[-1] == K, (x.shape, K)
    return x.numel() // K


def matvec_affine(w: AffineWeight, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    B = _rows(x, w.K)
    y = out if out is not None else torch.empty((B, w.N), dtype=torch.float16, device=x.device)
    check(lib().im_cuda_matvec_affine(w.handle, vp(x), vp(y), C.c_int(B), _stream()))
    return y


def silu_mul(gate: torch.Tensor, up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """silu_gate (crates/ironmill-inference/src/metal/shaders/activation/activation.metal): f16(SiLU(gate) * up), f32 inside."""
    assert gate.is_cuda and gate.dtype == torch.float16 and gate.is_contiguous() and up.shape == gate.shape and up.is_contiguous()
    y = out if out is not None else torch.empty_like(gate)
    check(lib().im_cuda_silu_mul(vp(gate), vp(up), vp(y), C.c_size_t(gate.numel()), _stream()))
    return y


def matmul_affine(w: AffineWeight, x: torch.Tensor, out: torch.Tensor | None = None, scratch: torch.Tensor | None = None) -> torch.Tensor:
    """Dense INT4 or INT8 g128 GEMM on the tensor cores (tcgen05; few tokens mma.sync): y[M, N] = f16(x / awq) @ dequant(w)^T.  scratch: M * K halves."""
    M = _rows(x, w.K)
    y = out if out is not None else torch.empty((M, w.N), dtype=torch.float16, device=x.device)
    if scratch is None:
        scratch = torch.empty((M, w.K), dtype=torch.float16, device=x.device)
    check(lib().im_cuda_matmul_affine(w.handle, vp(x), vp(y), C.c_int(M), vp(scratch), _stream()))
    return y


def matvec_affine_host(w: AffineWeight, x: np.ndarray) -> np.ndarray:
    x = np.ascontiguousarray(x)
    assert x.dtype == np.float16
    B = x.size // w.K
    y = np.empty((B, w.N), dtype=np.float16)
    check(lib().im_cuda_matvec_affine_host(w.handle, vp(x), vp(y), C.c_int(B)))
    return y


def ffn_gate_up_act(gate: AffineWeight, up: AffineWeight, x: torch.Tensor, out: torch.Tensor | None = None):
    B = _rows(x, gate.K)
    y = out if out is not None else torch.empty((B, gate.N), dtype=torch.float16, device=x.device)
    check(lib().im_cuda_ffn_gate_up_act(gate.handle, up.handle, vp(x), vp(y), C.c_int(B), _stream()))
    return y


def fused_residual_norm_matvec(w: AffineWeight, a: torch.Tensor, b: torch.Tensor, gamma: torch.Tensor, eps: float,
                               want_residual: bool = True, want_normed: bool = True):
    B = _rows(a, w.K)
    assert b.shape == a.shape and b.dtype == torch.float16 and gamma.dtype == torch.float16
    y = torch.empty((B, w.N), dtype=torch.float16, device=a.device)
    res = torch.empty_like(a) if want_residual else None
    nrm = torch.empty_like(a) if want_normed else None
    check(lib().im_cuda_fused_residual_norm_matvec(w.handle, vp(a), vp(b), vp(gamma), C.c_float(eps), vp(y), vp(res),
                                                   vp(nrm), C.c_int(B), _stream()))
    return y, res, nrm


def matvec_f16(w: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    assert w.is_cuda and w.dtype == torch.float16 and w.is_contiguous() and w.dim() == 2
    N, K = w.shape
    B = _rows(x, K)
    y = torch.empty((B, N), dtype=torch.float16, device=x.device)
    check(lib().im_cuda_matvec_f16(vp(w), vp(x), vp(y), C.c_int(N), C.c_int(K), C.c_int(B), _stream()))
    return y


# ---------------------------------------------------------------- norms / embedding / RoPE
def _h16(x):
    assert x.is_cuda and x.dtype == torch.float16 and x.is_contiguous()
    return x


def rms_norm(x: torch.Tensor, gamma: torch.Tensor, eps: float) -> torch.Tensor:
    H = x.shape[-1]
    out = torch.empty_like(_h16(x))
    check(lib().im_cuda_rms_norm(vp(x), vp(_h16(gamma)), vp(out), C.c_int(H), C.c_int(x.numel() // H), C.c_float(eps), _stream()))
    return out


def fused_residual_rms_norm(a, b, gamma, eps):
    H = a.shape[-1]
    normed, residual = torch.empty_like(_h16(a)), torch.empty_like(a)
    check(lib().im_cuda_fused_residual_rms_norm(vp(a), vp(_h16(b)), vp(_h16(gamma)), vp(normed), vp(residual), C.c_int(H),
                                                C.c_int(a.numel() // H), C.c_float(eps), _stream()))
    return normed, residual


def residual_add(a, b):
    out = torch.empty_like(_h16(a))
    check(lib().im_cuda_residual_add(vp(a), vp(_h16(b)), vp(out), C.c_size_t(a.numel()), _stream()))
    return out


def embedding_norm(tokens: torch.Tensor, table: torch.Tensor, gamma: torch.Tensor, eps: float, embed_scale: float = 1.0):
    assert tokens.is_cuda and tokens.dtype in (torch.int32, torch.uint32) and tokens.is_contiguous()
    vocab, H = _h16(table).shape
    T = tokens.numel()
    normed = torch.empty((T, H), dtype=torch.float16, device=table.device)
    raw = torch.empty_like(normed)
    check(lib().im_cuda_embedding_norm(vp(tokens), vp(table), vp(_h16(gamma)), vp(normed), vp(raw), C.c_int(H), C.c_int(T),
                                       C.c_uint32(vocab), C.c_float(eps), C.c_float(embed_scale), _stream()))
    return normed, raw


def rope_table(head_dim: int, max_pos: int, theta: float, rotary_dim: int | None = None, device="cuda"):
    cos = torch.empty((max_pos, head_dim // 2), dtype=torch.float16, device=device)
    sin = torch.empty_like(cos)
    check(lib().im_cuda_rope_table(C.c_int(head_dim), C.c_int(max_pos), C.c_double(theta), C.c_int(rotary_dim or 0), vp(cos), vp(sin)))
    return cos, sin


def qk_norm_rope_(q, k, qw, kw, cos, sin, nh, nkv, hd, seq_offset, eps, rotary_dim=None):
    """In place on q [T,nh,hd] and k [T,nkv,hd]."""
    T = _h16(q).numel() // (nh * hd)
    check(lib().im_cuda_qk_norm_rope(vp(q), vp(_h16(k)), vp(_h16(qw)), vp(_h16(kw)), vp(cos), vp(sin), C.c_int(nh), C.c_int(nkv),
                                     C.c_int(hd), C.c_int(rotary_dim or hd), C.c_int(seq_offset), C.c_int(T), C.c_float(eps), _stream()))


def rope_(qk, cos, sin, heads, hd, seq_offset):
    T = _h16(qk).numel() // (heads * hd)
    check(lib().im_cuda_rope(vp(qk), vp(cos), vp(sin), C.c_int(heads), C.c_int(hd), C.c_int(seq_offset), C.c_int(T), _stream()))


# ---------------------------------------------------------------- TurboQuant
def tq_lloyd_max(dim: int, n_bits: int):
    levels = np.zeros(1 << n_bits, dtype=np.float32)
    bounds = np.zeros((1 << n_bits) - 1, dtype=np.float32)
    check(lib().im_cuda_tq_lloyd_max(C.c_int(dim), C.c_int(n_bits), vp(levels), vp(bounds)))
    return levels, bounds


def tq_generate(head_dim: int, seed: int):
    signs = np.zeros(head_dim, dtype=np.float32)
    qjl = np.zeros((head_dim, head_dim), dtype=np.float32)
    check(lib().im_cuda_tq_generate(C.c_int(head_dim), C.c_uint64(seed), vp(signs), vp(qjl)))
    return signs, qjl


class TurboQuant:
    """MetalTurboQuantModel counterpart (crates/ironmill-inference/src/metal/turboquant/mod.rs:221-287)."""

    def __init__(self, dev: Device, head_dim: int, n_bits: int, signs: np.ndarray, qjl: np.ndarray,
                 k_levels=None, k_bounds=None, v_levels=None, v_bounds=None):
        self.dev, self.head_dim, self.n_bits = dev, head_dim, n_bits
        self.handle = C.c_void_p()
        f = lambda a: None if a is None else np.ascontiguousarray(a, dtype=np.float32)  # noqa: E731
        self._keep = [f(signs), f(qjl), f(k_levels), f(k_bounds), f(v_levels), f(v_bounds)]
        check(lib().im_cuda_tq_create(dev.handle, C.c_int(head_dim), C.c_int(n_bits), *[vp(a) for a in self._keep],
                                      C.byref(self.handle)))

    def encode(self, kv, is_k, cache, scale, r_norms, nkv, max_seq, base_pos, nseq=1, pos_dev=None):
        T = _h16(kv).numel() // (nseq * nkv * self.head_dim)
        check(lib().im_cuda_tq_encode(self.handle, vp(kv), C.c_int(int(is_k)), vp(cache), vp(scale), vp(r_norms), C.c_int(nseq),
                                      C.c_int(nkv), C.c_int(max_seq), C.c_int(base_pos), vp(pos_dev), C.c_int(T), _stream()))

    def attention(self, q, k_cache, v_cache, k_scale, v_scale, k_rnorm, attn_scale, nh, nkv, max_seq, base_pos, nseq=1,
                  pos_dev=None, num_splits=0):
        T = _h16(q).numel() // (nseq * nh * self.head_dim)
        out = torch.empty_like(q)
        check(lib().im_cuda_tq_attention(self.handle, vp(q), vp(k_cache), vp(v_cache), vp(k_scale), vp(v_scale), vp(k_rnorm),
                                         C.c_float(attn_scale), vp(out), C.c_int(nseq), C.c_int(nh), C.c_int(nkv), C.c_int(max_seq),
                                         C.c_int(base_pos), vp(pos_dev), C.c_int(T), C.c_int(num_splits), _stream()))
        return out

    def prefill_attention(self, q, k_cache, v_cache, k_scale, v_scale, k_rnorm, attn_scale, nh, nkv, max_seq, base_pos):
        """T tokens of one sequence at positions base_pos .. (rows already cached): dequantise once + causal tensor-core pass."""
        T = _h16(q).numel() // (nh * self.head_dim)
        out = torch.empty_like(q)
        dq = torch.empty(int(lib().im_cuda_tq_prefill_scratch_bytes(C.c_int(nkv), C.c_int(max_seq))), dtype=torch.uint8, device=q.device)
        check(lib().im_cuda_tq_prefill_attention(self.handle, vp(q), vp(k_cache), vp(v_cache), vp(k_scale), vp(v_scale), vp(k_rnorm),
                                                 C.c_float(attn_scale), vp(out), C.c_int(nh), C.c_int(nkv), C.c_int(max_seq), C.c_int(base_pos),
                                                 C.c_int(T), vp(dq), _stream()))
        return out

    def free(self):
        if self.handle:
            lib().im_cuda_tq_free(self.handle)
            self.handle = C.c_void_p()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def fused_residual_norm_ffn(gate: AffineWeight, up: AffineWeight, a, b, gamma, eps: float):
    """residual + RMSNorm + gate/up + SiLU in one launch -> (out [B, I], residual, normed)."""
    B = _rows(a, gate.K)
    out = torch.empty((B, gate.N), dtype=torch.float16, device=a.device)
    res, nrm = torch.empty_like(a), torch.empty_like(a)
    check(lib().im_cuda_fused_residual_norm_ffn(gate.handle, up.handle, vp(a), vp(_h16(b)), vp(_h16(gamma)), C.c_float(eps), vp(out),
                                                vp(res), vp(nrm), C.c_int(B), _stream()))
    return out, res, nrm


def tq_fused_attention(tq: "TurboQuant", qkv, nh, nkv, cos, sin, k_cache, v_cache, k_scale, v_scale, k_rnorm, attn_scale, max_seq,
                       base_pos, eps=1e-6, qw=None, kw=None, nseq=1, pos_dev=None, num_splits=0, rotary_dim=0):
    """(QK-norm +) RoPE + K/V cache write + attention from a fused QKV row [nseq*T, (nh + 2 nkv) * hd]."""
    hd = tq.head_dim
    stride = (nh + 2 * nkv) * hd
    MT = _h16(qkv).numel() // stride
    T = MT // nseq
    out = torch.empty((MT, nh * hd), dtype=torch.float16, device=qkv.device)
    qrot = torch.empty((MT, nh, 2, hd), dtype=torch.float32, device=qkv.device)
    check(lib().im_cuda_tq_fused_attention(tq.handle, vp(qkv), C.c_int(stride), C.c_int(nh * hd), C.c_int((nh + nkv) * hd), vp(qw), vp(kw),
                                           vp(cos), vp(sin), C.c_int(rotary_dim), C.c_float(eps), vp(k_cache), vp(v_cache), vp(k_scale),
                                           vp(v_scale), vp(k_rnorm), C.c_float(attn_scale), vp(qrot), vp(out), C.c_int(nseq), C.c_int(nh),
                                           C.c_int(nkv), C.c_int(max_seq), C.c_int(base_pos), vp(pos_dev), C.c_int(T), C.c_int(num_splits),
                                           _stream()))
    return out


def tq_attention_static(tq: "TurboQuant", q, k_cache, v_cache, k_scale, v_scale, k_rnorm, attn_scale, nh, nkv, max_seq, base_pos,
                        nseq=1, pos_dev=None, num_splits=0):
    """Attention through the entry point that allocates nothing (split partials in the library's built-in array)."""
    T = _h16(q).numel() // (nseq * nh * tq.head_dim)
    out = torch.empty_like(q)
    check(lib().im_cuda_tq_attention_static(tq.handle, vp(q), vp(k_cache), vp(v_cache), vp(k_scale), vp(v_scale), vp(k_rnorm),
                                            C.c_float(attn_scale), vp(out), C.c_int(nseq), C.c_int(nh), C.c_int(nkv), C.c_int(max_seq),
                                            C.c_int(base_pos), vp(pos_dev), C.c_int(T), C.c_int(num_splits), _stream()))
    return out


def kv_scatter_f16(proj, cache, nseq, T, nkv, max_seq, base_pos, pos_dev=None):
    """kv_scatter (shaders/kv/kv_scatter.metal:20-42): proj fp16 [nseq*T, nkv, 128] -> cache fp16 [nseq, nkv, max_seq, 128]."""
    check(lib().im_cuda_kv_scatter_f16(vp(proj), vp(cache), C.c_int(nseq), C.c_int(T), C.c_int(nkv), C.c_int(128), C.c_int(max_seq),
                                       C.c_int(base_pos), vp(pos_dev), None, _stream()))


def sdpa_f16(dev: "Device", q, k_cache, v_cache, scale, nh, nkv, max_seq, base_pos, nseq=1, pos_dev=None, num_splits=0):
    """fp16-KV attention (fused_sdpa / prefill_attention_v2 / fused_sdpa_split + reduce): q fp16 [nseq*T, nh, 128]."""
    T = _h16(q).numel() // (nseq * nh * 128)
    out = torch.empty_like(q)
    splits = num_splits if num_splits > 0 else 64
    nbytes = int(lib().im_cuda_sdpa_f16_scratch_bytes(C.c_int(nseq), C.c_int(T), C.c_int(nh), C.c_int(splits)))
    scratch = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=q.device)
    check(lib().im_cuda_sdpa_f16(dev.handle, vp(q), vp(k_cache), vp(v_cache), vp(out), C.c_int(nseq), C.c_int(nh), C.c_int(nkv), C.c_int(128),
                                 C.c_int(max_seq), C.c_int(base_pos), vp(pos_dev), C.c_int(T), C.c_float(scale), C.c_int(num_splits),
                                 vp(scratch), C.c_size_t(nbytes), _stream()))
    return out


# ---------------------------------------------------------------- KV cache in pages
_DTYPES = {torch.float16: IM_DTYPE_F16, torch.float32: IM_DTYPE_F32, torch.bfloat16: IM_DTYPE_BF16}


_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream  # a call here costs a tenth of torch.cuda's


def _launch(ordinal: int, fn, *args) -> None:
    """fn(*args, current stream) with the handle's device as the current one, as the C ABI asks for."""
    if _current_device() != ordinal:
        with torch.cuda.device(ordinal):
            return _launch(ordinal, fn, *args)
    check(fn(*args, _raw_stream(ordinal)))


def _rows_of(x: torch.Tensor, n: int, heads: int, dim: int, dtype, ordinal: int) -> int:
    """Elements between the tokens of x [n, heads, dim], whose heads lie side by side."""
    tokens, h, d = x.shape
    s, sh, sd = x.stride()
    assert tokens == n and h == heads and d == dim and x.dtype is dtype and x.get_device() == ordinal, (x.shape, x.dtype, x.device)
    assert sd == 1 and (sh == dim or h == 1), x.stride()
    return s if n > 1 else heads * dim


def _ints(x: torch.Tensor, ordinal: int, n: int, width: int = 0) -> int:
    """Address of int32 [n] or [n, width] in one piece."""
    assert x.dtype is torch.int32 and x.get_device() == ordinal and x.is_contiguous() and x.numel() == (n * width if width else n) and x.dim() == (2 if width else 1), \
        (x.dtype, x.shape, x.device)
    return x.data_ptr()


class PagedKV:
    """Keys and values of every layer in pages (im_paged_kv): k_pages, v_pages [layers, pages, kv_heads, page_size, head_dim] (fp16 or bf16; pages and
    layers may lie apart), page_table int32 [sequences, width], lengths int32 [sequences]: rows before a call's new tokens (a negative one
    counts as 0, one past the table as the table's rows). Holds the tensors; what is written to them is what the next call sees."""

    def __init__(self, dev: Device, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor):
        assert k_pages.is_cuda and k_pages.device.index == dev.ordinal and k_pages.dtype in (torch.float16, torch.bfloat16) and k_pages.dim() == 5
        assert v_pages.device == k_pages.device and v_pages.dtype == k_pages.dtype and v_pages.shape == k_pages.shape and v_pages.stride() == k_pages.stride()
        layers, pages, heads, page, dim = k_pages.shape
        s = k_pages.stride()
        assert s[4] == 1 and (page == 1 or s[3] == dim) and (heads == 1 or s[2] == page * dim), s
        assert (layers == 1 or s[0] > 0) and (pages == 1 or s[1] > 0), s  # an expanded axis would be taken for a packed one
        self.dev, self.k_pages, self.v_pages, self.ordinal = dev, k_pages, v_pages, dev.ordinal
        self.device, self.dtype, self.kv_heads, self.head_dim, self.layers = k_pages.device, k_pages.dtype, heads, dim, layers
        self.struct = PagedKvStruct(k_pages.data_ptr(), v_pages.data_ptr(), s[0] if layers > 1 else 0, s[1] if pages > 1 else 0, layers, pages, heads, page, dim,
                                    _DTYPES[k_pages.dtype])
        self.ref = C.addressof(self.struct)
        self.point_at(page_table, lengths)

    def point_at(self, page_table: torch.Tensor, lengths: torch.Tensor) -> None:
        """Another page table and other lengths, as paged_keep and paged_reorder return them."""
        assert page_table.dim() == 2 and page_table.dtype == torch.int32 and page_table.device == self.device
        n, width = page_table.shape
        assert (n == 0 or width == 1 or page_table.stride(1) == 1) and (n <= 1 or page_table.stride(0) >= width), page_table.stride()
        self.struct.seq_len_dev = _ints(lengths, self.ordinal, n)
        self.struct.num_seqs, self.struct.page_table_dev, self.struct.table_width = n, page_table.data_ptr(), width
        self.struct.table_stride = page_table.stride(0) if n > 1 else 0
        self.page_table, self.lengths, self.num_seqs = page_table, lengths, n
        self.scratch_bytes = {}  # of attention, by heads and new tokens


def paged_append(kv: PagedKV, layer: int, k, v, token_start, q=None, cos=None, sin=None, positions=None, rotary_dim=None, neighbours=False, q_out=None):
    """Keys and values [tokens, kv_heads, head_dim] of new tokens into the pages, keys and queries q [tokens, heads, head_dim] rotated on the
    way (returned in q_out, which may be q). token_start int32 [sequences + 1]; cos, sin [positions, head_dim / 2] fp16 or f32; positions
    int32 [tokens]: rows of the tables, where they are not the rows of the cache; neighbours: columns (2 i, 2 i + 1) belong together
    instead of the halves'. Without tables nothing is rotated."""
    n, dim, dtype, on = k.shape[0], kv.head_dim, kv.dtype, kv.ordinal
    ks, vs = _rows_of(k, n, kv.kv_heads, dim, dtype, on), _rows_of(v, n, kv.kv_heads, dim, dtype, on)
    heads = qs = qos = max_pos = table = 0
    qp = op = cp = sp = None
    if q is not None:
        heads = q.shape[1]
        qs, qp = _rows_of(q, n, heads, dim, dtype, on), q.data_ptr()
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            qos = heads * dim
        else:
            qos = _rows_of(q_out, n, heads, dim, dtype, on)
        op = q_out.data_ptr()
    else:
        assert q_out is None
    if cos is not None:
        max_pos, half = cos.shape
        assert sin.shape == cos.shape and half == dim // 2 and cos.dtype is sin.dtype and cos.is_contiguous() and sin.is_contiguous()
        assert cos.get_device() == on and sin.get_device() == on
        table, cp, sp = _DTYPES[cos.dtype], cos.data_ptr(), sin.data_ptr()
        rotary_dim = dim if rotary_dim is None else rotary_dim
    else:
        assert sin is None and not rotary_dim
        rotary_dim = 0
    _launch(on, lib().im_cuda_paged_append, kv.dev.handle, kv.ref, layer, k.data_ptr(), ks, v.data_ptr(), vs, _ints(token_start, on, kv.num_seqs + 1), n, qp, qs, op, qos,
            heads, cp, sp, table, max_pos, rotary_dim, 1 if neighbours else 0, None if positions is None else _ints(positions, on, n))
    return q_out


def _attention_bytes(kv: PagedKV, heads: int, max_new: int, max_len: int) -> int:
    key = (heads, max_new, max_len.bit_length())  # what is enough for the next power of two
    nbytes = kv.scratch_bytes.get(key)
    if nbytes is None:
        most = min(1 << max_len.bit_length(), 2 ** 31 - 1) if max_len else 0
        nbytes = kv.scratch_bytes[key] = int(lib().im_cuda_paged_attention_scratch_bytes(kv.dev.handle, kv.ref, heads, max_new, most))
    return nbytes


def paged_attention_scratch(kv: PagedKV, heads: int, max_new: int, max_len: int = 0) -> torch.Tensor:
    """Scratch for paged_attention calls of this cache with so many heads, new tokens and rows (or fewer rows); calls that may overlap need
    one each."""
    return torch.empty(max(_attention_bytes(kv, heads, max_new, max_len), 16), dtype=torch.uint8, device=kv.device)


def paged_attention(kv: PagedKV, layer: int, q, token_start, max_new: int, scale: float, mask=None, max_len=0, out=None, scratch=None):
    """softmax(scale * q K^T) V of new tokens q [tokens, heads, head_dim] whose rows are in the pages: every token sees the `lengths` rows before
    the new ones and, without a mask, its own and the new ones before it; with mask int64 [tokens, words] the new ones whose bits
    are set (of a drafted tree: its ancestors and itself). max_new, max_len: the most new tokens and rows of a sequence."""
    n, heads, dim = q.shape
    on = kv.ordinal
    qs = _rows_of(q, n, heads, kv.head_dim, kv.dtype, on)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os_ = heads * dim
    else:
        os_ = _rows_of(out, n, heads, dim, kv.dtype, on)
    words, mp = 0, None
    if mask is not None:
        rows, words = mask.shape
        assert mask.dtype is torch.int64 and rows == n and mask.is_contiguous() and mask.get_device() == on
        mp = mask.data_ptr()
    nbytes, at = 0, None
    if scratch is None:
        nbytes = _attention_bytes(kv, heads, max_new, max_len)
        if nbytes:
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=kv.device)
            at = scratch.data_ptr()
    else:
        assert scratch.dtype is torch.uint8 and scratch.get_device() == on and scratch.is_contiguous()
        nbytes, at = scratch.numel(), scratch.data_ptr()
    _launch(on, lib().im_cuda_paged_attention, kv.dev.handle, kv.ref, layer, q.data_ptr(), qs, out.data_ptr(), os_, heads, _ints(token_start, on, kv.num_seqs + 1), n, max_new,
            mp, words, scale, max_len, at, nbytes)
    return out


def paged_keep(kv: PagedKV, accepted, counts, lengths_out=None):
    """The accepted path of every drafted tree, accepted int32 [sequences, most] (places among the new rows, from the root on), counts int32
    [sequences], moves up behind the rows before it, in every layer. Returns the new lengths (kv.point_at)."""
    most, n, on = accepted.shape[1], kv.num_seqs, kv.ordinal
    if lengths_out is None:
        lengths_out = torch.empty_like(kv.lengths)
    _launch(on, lib().im_cuda_paged_keep, kv.dev.handle, kv.ref, _ints(accepted, on, n, most), most, _ints(counts, on, n), _ints(lengths_out, on, n))
    return lengths_out


def paged_reorder(kv: PagedKV, parents, group: int, table_out=None, lengths_out=None):
    """Beam i of every group of sequences becomes a copy of beam parents[i] (int32 [sequences]): pages are shared up to the last one, whose rows
    are copied where a parent has several children, into the pages of a beam that has none. From its last page on a row's pages are its own. Returns the new page table and lengths (kv.point_at)."""
    n, width = kv.page_table.shape
    on = kv.ordinal
    if table_out is None:
        table_out, stride = kv.page_table.new_empty((n, width)), width
    else:
        assert table_out.shape == (n, width) and table_out.dtype is torch.int32 and table_out.get_device() == on and (n == 0 or width == 1 or table_out.stride(1) == 1)
        assert n <= 1 or table_out.stride(0) >= width, table_out.stride()
        stride = table_out.stride(0) if n > 1 else 0
    if lengths_out is None:
        lengths_out = torch.empty_like(kv.lengths)
    _launch(on, lib().im_cuda_paged_reorder, kv.dev.handle, kv.ref, _ints(parents, on, n), group, table_out.data_ptr(), stride, _ints(lengths_out, on, n))
    return table_out, lengths_out


# ---------------------------------------------------------------- beam search
def beam_select_scratch(dev: Device, groups: int, beams: int, vocab: int, picks: int) -> torch.Tensor:
    """Scratch for beam_select calls of these sizes; calls that may overlap need one each."""
    return torch.empty(max(_select_bytes(dev, (groups, beams, vocab, picks)), 16), dtype=torch.uint8, device=dev.torch_device)


def _select_bytes(dev: Device, key) -> int:
    nbytes = dev.select_bytes.get(key)
    if nbytes is None:
        nbytes = dev.select_bytes[key] = int(lib().im_cuda_beam_select_scratch_bytes(dev.handle, *key))
    return nbytes


def beam_select(dev: Device, logits, scores, picks: int, done=None, end_token=-1, scratch=None):
    """The `picks` best of score + log_softmax(logits) over beams and vocabulary: logits [groups, beams, vocab] (fp16, bf16 or f32), scores f32
    [groups, beams], done bool [groups, beams]. Returns scores f32, parents and tokens int32 [groups, picks], best first, ties to
    the lowest beam and token; a finished beam has one continuation, end_token at its own score."""
    groups, beams, vocab = logits.shape
    on, (sg, sb, sv) = dev.ordinal, logits.stride()
    assert logits.get_device() == on and (sv == 1 or vocab == 1) and (groups == 1 or beams == 1 or sg == beams * sb), logits.stride()
    stride = (sb if beams > 1 else sg) if groups * beams > 1 else 0
    assert groups * beams <= 1 or stride >= vocab, logits.stride()  # rows in common would be taken for packed ones
    assert scores.shape == (groups, beams) and scores.dtype is torch.float32 and scores.is_contiguous() and scores.get_device() == on
    dp = None
    if done is not None:
        assert done.shape == (groups, beams) and done.dtype in (torch.bool, torch.uint8) and done.is_contiguous() and done.get_device() == on
        dp = done.data_ptr()
    nbytes, at = 0, None
    if scratch is None:
        nbytes = _select_bytes(dev, (groups, beams, vocab, picks))
        if nbytes:
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev.torch_device)
            at = scratch.data_ptr()
    else:
        assert scratch.dtype is torch.uint8 and scratch.get_device() == on and scratch.is_contiguous()
        nbytes, at = scratch.numel(), scratch.data_ptr()
    score = scores.new_empty((groups, picks))
    parent = torch.empty_like(score, dtype=torch.int32)
    token = torch.empty_like(parent)
    _launch(on, lib().im_cuda_beam_select, dev.handle, logits.data_ptr(), _DTYPES[logits.dtype], stride, groups, beams, vocab,
            scores.data_ptr(), dp, end_token, picks, score.data_ptr(), parent.data_ptr(), token.data_ptr(), at, nbytes)
    return score, parent, token
