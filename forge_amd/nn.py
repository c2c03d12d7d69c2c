"""PyTorch modules of the INT8 path, shaped like the reference's python/forge/nn/linear.py:115-254.

QuantizedLinear and SparseLinear keep the reference's parameter and buffer names, shapes and
dtypes:
- QuantizedLinear: w_int8 (N, K) int8 buffer, w_scale (N) fp16, bias (N) fp16 or None;
- SparseLinear: W_comp (N, K/2) int8 buffer, w_meta (N, K/32) int32 buffer, w_scale, bias.
The one stored difference is the order of the 2:4 index words in w_meta: here the gfx950 SMFMAC
order (forge_pack_metadata), in the reference the row-major order (pack_metadata.cu:23-29); the
word values and the raw nibbles are the same. SparseLinear's state_dict carries layout version 2
in its metadata (torch's per-module `version`); load_state_dict converts w_meta from the
reference order when the version is lower or absent (a reference checkpoint: the reference
module has torch's default version 1), so a reference state_dict loads as is and computes the
reference's outputs. w_meta_from_reference / w_meta_to_reference convert a whole tensor on any
device.

Forward runs the library (forge_int8_linear / forge_sparse_int8_linear); there is no other path.

Without a counterpart in the reference: Int4Linear (4-bit weights with group scales, for the few tokens of a
decode step) and DecoderAttention (the attention block of a decoder on it: projection, norm and rotation of the heads,
attention over prompts or over a paged cache). Both serve only: no backward.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn
from torch.autograd import forward_ad

from . import ops


def _prep_device(module_tensor: torch.Tensor) -> torch.device:
    """Weight preparation runs on the module's device, or cuda:0 for a CPU module."""
    return module_tensor.device if module_tensor.is_cuda else torch.device("cuda", 0)


def _as_weight(weight_fp: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """The reference converts any float weight to float32 (linear.py:169, :234); fp16 and fp32
    go to the device as they are (the kernel widens fp16 exactly), other dtypes as float32."""
    w = weight_fp if weight_fp.dtype in (torch.float16, torch.float32) else weight_fp.to(torch.float32)
    return w.to(dev).contiguous()


def _plain(*tensors: torch.Tensor) -> bool:
    """Whether a foreign call on the tensors' addresses can stand for torch operators on them: no
    tensor without memory of its own (batched gradients, zero tensors, fake and other subclasses), no
    dispatch mode that has to see the operators (tracing), no forward-mode tangents."""
    if torch._C._len_torch_dispatch_stack() or forward_ad._current_level >= 0:
        return False
    for t in tensors:
        if type(t) not in (torch.Tensor, nn.Parameter) or not torch._C._has_storage(t) or t._is_zerotensor():
            return False
    return True


class _Int8LinearFn(torch.autograd.Function):
    """Forward on the INT8 path; backward through the dequantized FP16 weight, returning the
    input and bias gradients (the reference's _Int8LinearFn, linear.py:115-132)."""

    @staticmethod
    def forward(ctx, x, w_int8, w_scale, bias, scratch_a, scratch_s):
        ctx.save_for_backward(w_int8, w_scale)
        ctx.has_bias = bias is not None
        return ops.int8_linear(x, w_int8, w_scale, bias, scratch_a, scratch_s)

    @staticmethod
    def backward(ctx, grad_output):
        w_int8, w_scale = ctx.saved_tensors
        g = grad_output if grad_output.dtype == torch.float16 else grad_output.to(torch.float16)
        # With gradients recorded (create_graph=True), batched or traced the torch operators below
        # carry them; the library's passes would not. Saved-tensor hooks may have changed layouts and
        # devices. The library sums whole FP16 vectors of a non-empty batch.
        if (not torch.is_grad_enabled() and grad_output.dtype == torch.float16 and _plain(g, w_int8, w_scale)
                and g.is_cuda and w_int8.device == g.device and w_scale.device == g.device and w_int8.is_contiguous()
                and w_scale.is_contiguous() and w_scale.dtype == torch.float16 and g.shape[0] > 0 and g.shape[1] >= 8):
            if not g.is_contiguous():
                g = g.contiguous()
            w16, grad_bias = ops.int8_linear_backward_prep(w_int8, w_scale, g, ctx.has_bias)
            return g @ w16, None, None, grad_bias, None, None
        w16 = w_int8.to(torch.float16) * w_scale.unsqueeze(1)
        grad_x = g @ w16
        grad_bias = grad_output.sum(dim=0).to(torch.float16) if ctx.has_bias else None
        return grad_x, None, None, grad_bias, None, None


class QuantizedLinear(nn.Module):
    """INT8 linear layer: y = dequant(quantize_per_token(x) @ w_int8^T) + bias, FP16 in and out
    (linear.py:135-184)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True):
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.register_buffer("w_int8", torch.zeros(out_features, in_features, dtype=torch.int8))
        self.w_scale = nn.Parameter(torch.ones(out_features, dtype=torch.float16))
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features, dtype=torch.float16))
        else:
            self.register_parameter("bias", None)
        self._scratch_a: Optional[torch.Tensor] = None
        self._scratch_s: Optional[torch.Tensor] = None

    def _scratch(self, M: int, K: int, device):
        a = self._scratch_a
        if a is None or a.shape[0] < M or a.shape[1] != K or a.device != device:
            self._scratch_a = torch.empty(M, K, dtype=torch.int8, device=device)
            self._scratch_s = torch.empty(M, dtype=torch.float32, device=device)
        return self._scratch_a[:M], self._scratch_s[:M]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        M, K = x.shape
        a, s = self._scratch(M, K, x.device)
        return _Int8LinearFn.apply(x, self.w_int8, self.w_scale, self.bias, a, s)

    @torch.no_grad()
    def quantize_weight(self, weight_fp: torch.Tensor) -> None:
        """Per-output-row symmetric quantization (linear.py:167-173) on the device:
        scale = max(amax|w|, 1e-8) / 127, w_int8 = clamp(round(w / scale), -127, 127) (round half
        to even, IEEE division), scale stored as FP16."""
        q, scale = ops.quantize_weight_rows(_as_weight(weight_fp, _prep_device(self.w_int8)))
        self.w_int8.copy_(q)
        self.w_scale.data.copy_(scale)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


class _SparseInt8LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W_comp, w_meta, w_scale, bias, scratch_q, scratch_s):
        # split_k = 0: the planner's automatic tile and split, as the reference module asks
        # (linear.py:191-193); every plan gives the same bits.
        return ops.sparse_int8_linear(x, W_comp, w_meta, w_scale, bias, scratch_q, scratch_s, split_k=0)

    @staticmethod
    def backward(ctx, grad_output):
        raise NotImplementedError("SparseLinear has no backward (as in the reference, linear.py:201-203)")


class SparseLinear(nn.Module):
    """2:4 structured-sparse INT8 linear layer (linear.py:206-254). in_features % 64 == 0 and
    out_features % 16 == 0.

    State-dict layout version 2: w_meta in the gfx950 word order. Loading a state_dict whose
    metadata says version 1 or nothing (the reference's own modules save version 1) converts
    w_meta from the reference's row-major order first."""

    _version = 2

    def __init__(self, in_features: int, out_features: int, bias: bool = True):
        super().__init__()
        if in_features % 64 != 0 or out_features % 16 != 0:
            raise ValueError("SparseLinear needs in_features % 64 == 0 and out_features % 16 == 0")
        self.in_features = in_features
        self.out_features = out_features
        self.register_buffer("W_comp", torch.zeros(out_features, in_features // 2, dtype=torch.int8))
        self.register_buffer("w_meta", torch.zeros(out_features, in_features // 32, dtype=torch.int32))
        self.w_scale = nn.Parameter(torch.ones(out_features, dtype=torch.float16))
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features, dtype=torch.float16))
        else:
            self.register_parameter("bias", None)
        self._scratch_q: Optional[torch.Tensor] = None
        self._scratch_s: Optional[torch.Tensor] = None

    def _scratch(self, M: int, K: int, device):
        q = self._scratch_q
        if q is None or q.shape[0] < M or q.shape[1] != K or q.device != device:
            self._scratch_q = torch.empty(M, K, dtype=torch.int8, device=device)
            self._scratch_s = torch.empty(M, dtype=torch.float32, device=device)
        return self._scratch_q[:M], self._scratch_s[:M]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        M, K = x.shape
        q, s = self._scratch(M, K, x.device)
        return _SparseInt8LinearFn.apply(x, self.W_comp, self.w_meta, self.w_scale, self.bias, q, s)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                              error_msgs):
        version = local_metadata.get("version", None) if local_metadata else None
        key = prefix + "w_meta"
        if (version is None or version < 2) and key in state_dict:
            meta = state_dict[key]
            if meta.dim() != 2 or meta.shape[1] * 32 != self.in_features or meta.shape[0] != self.out_features:
                error_msgs.append(f"{key}: expected a ({self.out_features}, {self.in_features // 32}) tensor of the "
                                  f"reference's index words, got {tuple(meta.shape)}")
                return
            state_dict = dict(state_dict)
            state_dict[key] = w_meta_from_reference(meta.to(torch.int32))
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                                      error_msgs)

    @torch.no_grad()
    def from_dense_weight(self, weight_fp: torch.Tensor) -> None:
        """linear.py:231-249 in one device pass (forge_prepare_sparse_weight): quantize per row
        as QuantizedLinear does, prune 2:4 (the lower-magnitude pair of each group of 4),
        compress, and write the index words in the gfx950 order."""
        comp, meta, scale = ops.prepare_sparse_weight(_as_weight(weight_fp, _prep_device(self.W_comp)))
        self.W_comp.copy_(comp)
        self.w_meta.copy_(meta)
        self.w_scale.data.copy_(scale)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, sparse=2:4")


class _Int4LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_int4, w_scale, bias):
        return ops.int4_linear(x, w_int4, w_scale, bias)

    @staticmethod
    def backward(ctx, grad_output):
        raise NotImplementedError("Int4Linear has no backward")


class Int4Linear(nn.Module):
    """Linear layer with 4-bit weights and an FP16 scale per group_size (32, 64 or 128) values of a row:
    y = x @ (q * scale)^T + bias, x of `dtype` (float16 or bfloat16), FP32 sums (ops.int4_linear)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, group_size: int = 128,
                 dtype: torch.dtype = torch.float16):
        super().__init__()
        if group_size not in (32, 64, 128) or in_features % group_size != 0:
            raise ValueError("Int4Linear needs group_size 32, 64 or 128 and in_features % group_size == 0")
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"dtype must be torch.float16 or torch.bfloat16, got {dtype}")
        self.in_features = in_features
        self.out_features = out_features
        self.group_size = group_size
        # 0x88: eight weights of zero
        self.register_buffer("w_int4", torch.full((out_features, ops.int4_row_bytes(in_features)), 0x88, dtype=torch.uint8))
        self.register_buffer("w_scale", torch.ones((out_features, in_features // group_size), dtype=torch.float16))
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features, dtype=dtype))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = _Int4LinearFn.apply(x.reshape(-1, self.in_features), self.w_int4, self.w_scale, self.bias)
        return y.view(*x.shape[:-1], self.out_features)

    @torch.no_grad()
    def quantize_weight(self, weight_fp: torch.Tensor) -> None:
        """Symmetric quantization of each group of a row on the device (ops.quantize_weight_int4)."""
        q, scale = ops.quantize_weight_int4(_as_weight(weight_fp, _prep_device(self.w_int4)), self.group_size)
        self.w_int4.copy_(q)
        self.w_scale.copy_(scale)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"group_size={self.group_size}")


def tree_masks(parents: torch.Tensor) -> torch.Tensor:
    """ops.cache_attention's tree of drafted tokens from each token's parent, (B, T) integers on the host: -1 for a
    token that follows the cache, else an earlier token of its row. Token t sees itself, its parent, and so on."""
    if parents.dim() != 2 or not 1 <= parents.shape[1] <= 64:
        raise ValueError(f"parents must be (B, 1 to 64), got {tuple(parents.shape)}")
    rows = []
    for row in parents.tolist():
        masks = []
        for t, p in enumerate(row):
            if not -1 <= p < t:
                raise ValueError(f"token {t}'s parent must be -1 or an earlier token, got {p}")
            masks.append((1 << t) | (masks[p] if p >= 0 else 0))
        rows.append([m - (1 << 64) if m >> 63 else m for m in masks])
    return torch.tensor(rows, dtype=torch.int64)


class DecoderAttention(nn.Module):
    """The attention block of a decoder: one 4-bit projection to queries, keys and values, RMS norm and rotation of
    the query and key heads, attention, and the 4-bit output projection.

    Keys and values live in a paged cache of the caller's, (pages, page size, kv_heads, head_dim) each; `slots` says
    where each token's go (page * page size + offset)."""

    def __init__(self, hidden: int, heads: int, kv_heads: int, head_dim: int, positions: int, group_size: int = 128,
                 theta: float = 10000.0, eps: float = 1e-6, dtype: torch.dtype = torch.float16):
        super().__init__()
        if heads % kv_heads != 0 or head_dim % 16 != 0 or head_dim > 256:
            raise ValueError("DecoderAttention needs heads % kv_heads == 0 and a head_dim of a multiple of 16 up to 256")
        self.heads, self.kv_heads, self.head_dim, self.eps = heads, kv_heads, head_dim, eps
        self.qkv = Int4Linear(hidden, (heads + 2 * kv_heads) * head_dim, False, group_size, dtype)
        self.out = Int4Linear(heads * head_dim, hidden, False, group_size, dtype)
        self.q_norm = nn.Parameter(torch.ones(head_dim, dtype=dtype), requires_grad=False)
        self.k_norm = nn.Parameter(torch.ones(head_dim, dtype=dtype), requires_grad=False)
        # in 64 bits: FP32 angles of 130 thousand positions are off by up to 0.008
        angle = torch.arange(positions)[:, None] * theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
        self.register_buffer("cos", angle.cos().float(), persistent=False)
        self.register_buffer("sin", angle.sin().float(), persistent=False)

    def _heads(self, x):
        """The projections of (tokens, hidden): views of queries, keys and values in one output."""
        return self.qkv(x).view(x.shape[0], -1, self.head_dim).split((self.heads, self.kv_heads, self.kv_heads), 1)

    @torch.no_grad()
    def prompt(self, x: torch.Tensor, cu_seqlens: torch.Tensor, positions: torch.Tensor, k_cache: torch.Tensor,
               v_cache: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
        """Whole prompts packed into x (tokens, hidden), sequence b being tokens cu_seqlens[b] to cu_seqlens[b + 1] - 1; their
        keys and values go into the cache too."""
        q, k, v = self._heads(x)
        keys = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        q = ops.qk_norm_rope_cache(q, k, v, self.q_norm, self.k_norm, self.cos, self.sin, positions, k_cache, v_cache, slots,
                                   eps=self.eps, k_out=keys)
        return self.out(ops.prompt_attention(q, keys, v, cu_seqlens).view(x.shape[0], -1))

    @torch.no_grad()
    def cached(self, x: torch.Tensor, positions: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
               slots: torch.Tensor, page_table: torch.Tensor, cache_lens: torch.Tensor,
               tree: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The newest T tokens of each sequence, x (B, T, hidden), over the cache: one token, or a tree of drafts
        (tree_masks). positions and slots are (B * T,); token t of sequence b is at cache position cache_lens[b] + t."""
        B, T, hidden = x.shape
        q, k, v = self._heads(x.reshape(B * T, hidden))
        q = ops.qk_norm_rope_cache(q, k, v, self.q_norm, self.k_norm, self.cos, self.sin, positions, k_cache, v_cache, slots,
                                   eps=self.eps)
        o = ops.cache_attention(q.view(B, T, self.heads, self.head_dim), k_cache, v_cache, page_table, cache_lens, tree)
        return self.out(o.view(B, T, -1))


def _gfx950_word_positions(N: int, W: int, device) -> torch.Tensor:
    """Position in the gfx950 layout of reference word (n, c) (row-major index n * W + c):
    (n / 16) * W * 16 + c * R + n % 16, R = the rows of n's 16-row block (16, or fewer in a
    ragged last block), as forge_pack_metadata stores them."""
    n = torch.arange(N, device=device, dtype=torch.int64).unsqueeze(1)
    c = torch.arange(W, device=device, dtype=torch.int64).unsqueeze(0)
    blk = n // 16
    rows = torch.clamp(N - 16 * blk, max=16)
    return (blk * W * 16 + c * rows + n % 16).reshape(-1)


def w_meta_from_reference(w_meta_ref: torch.Tensor) -> torch.Tensor:
    """The reference's (N, K/32) int32 index words (word (n, c) = sum_g nib[n, 8c+g] << 4g,
    pack_metadata.cu:23-29) -> the same words in the gfx950 order, on the tensor's device."""
    N, W = w_meta_ref.shape
    src = w_meta_ref.contiguous().view(torch.int32).reshape(-1)
    out = torch.empty(N * W, dtype=torch.int32, device=src.device)
    out[_gfx950_word_positions(N, W, src.device)] = src
    return out.view(N, W)


def w_meta_to_reference(w_meta: torch.Tensor) -> torch.Tensor:
    """Inverse of w_meta_from_reference: gfx950-order words -> the reference's row-major words."""
    N, W = w_meta.shape
    src = w_meta.contiguous().view(torch.int32).reshape(-1)
    return src[_gfx950_word_positions(N, W, src.device)].view(N, W).clone()
