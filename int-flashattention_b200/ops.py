"""Python operator surface over libintfa.so, mirroring the reference's operators.

    attention_full_int8(q, k, v, q_scale, k_scale, v_scale, causal, sm_scale) -> o
        (flash_atten_full_int8.py:187,223)
    attention_int8(q, k, v, q_scale, k_scale, causal, sm_scale) -> o
        (flash_atten_int8.py:181,217)
    quant_pertoken / quant_pertensor (benchmark.py:96-107) and quant_perchannel
    int_flash_attention(q16, k16, v16, causal, sm_scale, variant): prologue + forward

Positional arguments and their meaning are the reference's.  Tensors must live on a
CUDA device; launches are asynchronous on torch's current stream of that device.
PyTorch is used for memory and streams only -- every computation runs in libintfa.so, and there is no other path: a
missing library or a CPU tensor raises.  Argument checks, allocation and launches are native code (csrc/intfa_torch.cpp,
module _native); the functions here give them their signatures.
"""
import math

import torch

from . import _lib

_native_mod = None


def _native():
    """The binding, loaded on first use (this package must be importable before it is built)."""
    global _native_mod
    if _native_mod is None:
        _lib.load()
        try:
            from . import _native as mod
        except ImportError as e:
            raise RuntimeError("_native.so is not built (or not for this Python): build it with `python "
                               "int-flashattention_b200/build.py`; there is no non-CUDA fallback. (%s)" % e) from e
        mod.set_error_class(_lib.IntfaError)
        _native_mod = mod
    return _native_mod


def default_G(head_dim, variant="full"):
    """Running-max granularity used when the caller does not choose one.  full-int8: the widest KV
    tile the reference's kernels allow for this head size (BLOCK_N <= HEAD_DIM,
    flash_atten_full_int8.py:88).  half-int8: 128 -- its result does not depend on G beyond fp16
    rounding, and 128-wide KV tiles are the faster ones at both head sizes."""
    if variant == "half":
        return 64 if head_dim == 256 else 128      # (fp16 V tiles of 128 keys x 256 channels do not fit next to K)
    return 128 if head_dim >= 128 else (64 if head_dim >= 64 else 32)


def _status_word(dev):
    """The int32[1] tensor of a device that the kernels report bounded-wait expiry into."""
    return _native().status(dev.index if dev.index is not None else torch.cuda.current_device())


def check_status(device=None):
    """Synchronise and raise if any kernel launched through this module on `device` gave up a
    bounded device-side wait, or was given a position, length or page outside its table or cache.  Returns the raw status word (0 = fine)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    word = _status_word(dev)
    val = int(word.item())
    if val != 0:
        word.zero_()
        if val & 0xff == _lib.STATUS_BAD_INDEX:
            raise _lib.IntfaError(_lib.ERR_INVALID_ARG, "a position, length or page lies outside its table or cache (nothing was read or written there)")
        raise _lib.IntfaError(_lib.ERR_DEVICE_WAIT,
                              "device-side wait expired (wait code %d, CTA %d)" % (val & 0xff, val >> 8))
    return val


def _fwd(variant, q, k, v, q_scale, k_scale, v_scale, causal, sm_scale, **kw):
    """The forward.  Keyword arguments: G, p_round, kv_order, state, q_offset, kv_offset, return_state, return_lse, write_o,
    debug_tap, out_dtype, debug_wait (test hooks of the bounded waits: (limit in kilo-cycles, K step to leave out))."""
    return (_native_mod or _native()).fwd(variant == "full", q, k, v, q_scale, k_scale, v_scale, causal, sm_scale, **kw)


def attention_full_int8(q, k, v, q_scale, k_scale, v_scale, causal, sm_scale, **kw):
    """Full-int8 attention forward (int8 Q/K/V, int8 P).  Mirrors attention_full_int8 of
    flash_atten_full_int8.py:187,223.  With causal=True the running maximum is carried from the
    off-band to the on-band stage (as flash_atten_int8.py:66,157,166 does); the reference's
    full-int8 Triton kernel drops it (flash_atten_full_int8.py:71,166-179).
    Extra keyword arguments (not in the reference): G (running-max granularity, the reference's
    BLOCK_N), p_round ("triton" | "rne"), kv_order ("ascending" | "descending": the CUDA path walks the KV tiles
    last to first, csrc/flash_fwd_kernel_full_qi8.h:331-469), v_scale of shape (B,H,ceil(Nk/G),D) (one row per KV
    tile, the CUDA path's layout), state/q_offset/kv_offset/return_state (ring attention),
    return_lse, debug_tap, out_dtype (torch.float16 | torch.bfloat16).  k, v and their scales may have
    fewer heads than q (grouped-query attention: query head h reads K/V head h // (H // H_kv))."""
    return (_native_mod or _native()).fwd(True, q, k, v, q_scale, k_scale, v_scale, causal, sm_scale, **kw)


def attention_int8(q, k, v, q_scale, k_scale, causal, sm_scale, **kw):
    """Half-int8 attention forward (int8 Q/K, fp16 V and P).  Mirrors attention_int8 of
    flash_atten_int8.py:181,217.  V may also be torch.float8_e5m2: P is then cast to e5m2 as well and P V runs as an
    fp8 matrix product with fp32 accumulation (flash_atten_int8.py:55-56,160)."""
    return (_native_mod or _native()).fwd(False, q, k, v, q_scale, k_scale, None, causal, sm_scale, **kw)


# ---------------------------------------------------------------------------------------------
# quantisation prologue
# ---------------------------------------------------------------------------------------------
def quant_pertoken(X):
    """benchmark.py:96-100.  Returns (int8 [B,H,N,D], scale [B,H,N]); the scale is fp32 holding
    the reference's fp16 value."""
    return (_native_mod or _native()).quant_pertoken(X)


def quant_qkv(q, k, v=None, v_mode="per_channel"):
    """The quantisation prologue of one attention call in one or two launches (one when v is None): per-token q and k
    (benchmark.py:96-100), and v (benchmark.py:102-107 or its per-channel form) with them, or after them where the call is
    larger; where v takes two passes the first, its column absmax, is in the grid of q and k.  Bit-identical to quant_pertoken / quant_perchannel / quant_pertensor called one by one.
    Returns (q8, q_scale, k8, k_scale) and, with v, (v8, v_scale) appended."""
    return (_native_mod or _native()).quant_qkv(q, k, v, _lib.VSCALE_PER_CHANNEL if v_mode == "per_channel" else _lib.VSCALE_PER_TENSOR)


def quant_v_with_allreduce(X, mode, group=None):
    """V quantisation for a token-sharded V: local column absmax, all-reduce(MAX) over `group`
    of the B*H*D fp32 bit patterns (order-preserving as int32 because they are non-negative),
    then the quantising pass.  Equals quantising the unsharded tensor bit for bit."""
    import ctypes
    import torch.distributed as dist
    lib = _lib.load()
    if not X.is_cuda:
        raise RuntimeError("int-flashattention_b200 runs on CUDA tensors only (there is no CPU path)")
    if X.dtype != torch.float16 or X.dim() != 4:
        raise TypeError("quantisers take a float16 [B,H,N,D] tensor")
    if X.stride(-1) != 1 or X.data_ptr() % 16 or any(s % 8 for s in X.stride()[:3]):
        X = X.contiguous()
    stream = ctypes.c_void_p(torch.cuda.current_stream(X.device).cuda_stream)
    B, H, N, D = X.shape
    mode_i = {"per_channel": _lib.VSCALE_PER_CHANNEL, "per_tensor": _lib.VSCALE_PER_TENSOR}.get(mode, mode)
    colmax = torch.zeros(B * H * D, dtype=torch.int32, device=X.device)
    st = _lib._i64x3(*X.stride()[:3])
    with torch.cuda.device(X.device):
        _lib.check(lib.intfa_v_colmax(X.data_ptr(), st, colmax.data_ptr(), B, H, N, D, stream))
    if dist.is_initialized() and dist.get_world_size(group) > 1:
        dist.all_reduce(colmax, op=dist.ReduceOp.MAX, group=group)
    x8 = torch.empty((B, H, N, D), dtype=torch.int8, device=X.device)
    shape = (B, H, D) if mode_i == _lib.VSCALE_PER_CHANNEL else (B, H)
    scale = torch.empty(shape, dtype=torch.float32, device=X.device)
    with torch.cuda.device(X.device):
        _lib.check(lib.intfa_v_quant_from_colmax(X.data_ptr(), st, colmax.data_ptr(), x8.data_ptr(),
                                                 scale.data_ptr(), mode_i, B, H, N, D, stream))
    return x8, scale


def quant_pertensor(X):
    """benchmark.py:102-107: one scale per (batch, head).  Returns (int8, scale [B,H] fp32)."""
    return (_native_mod or _native()).quant_v(X, _lib.VSCALE_PER_TENSOR)


def quant_perchannel(X):
    """Per-channel V quantisation: one scale per (batch, head, channel). Returns (int8, scale [B,H,D] fp32)."""
    return (_native_mod or _native()).quant_v(X, _lib.VSCALE_PER_CHANNEL)


def int_flash_attention(q, k, v, causal, sm_scale, variant="full", v_mode="per_channel", **kw):
    """fp16 Q/K/V in, fp16 O out: fused quantisation prologue (per-token Q/K; per-channel or
    per-(batch,head) V for the full-int8 variant) followed by the INT8 attention forward.
    Argument order follows the reference's attention(q, k, v, causal, sm_scale) (flash_atten_fp.py:155)."""
    return (_native_mod or _native()).flash(q, k, v, causal, sm_scale, variant, v_mode, **kw)


# ---------------------------------------------------------------------------------------------
# serving: rotary positions, a paged int8 cache, attention over it
# ---------------------------------------------------------------------------------------------
def rotary_table(n, rot_dim, base=10000.0, *, scaling=None, device=None):
    """(cos, sin) of positions 0 .. n-1 for the first `rot_dim` channels of a head: float32 [n, rot_dim/2, 2], from angles
    position * base**(-2j/rot_dim) in 64 bits.  `scaling` for contexts longer than those trained on:
      ("linear", factor)     every position divided by factor
      ("ntk", factor)        the base raised to base * factor**(rot_dim/(rot_dim-2)): the slowest pair turns factor times slower,
                             the fastest as before
      ("by_parts", factor, trained[, fast=32, slow=1[, magnitude]])
                             pairs that turn more than `fast` times within the `trained` positions stay, those that turn fewer
                             than `slow` times are divided by factor, in between by a ramp over the logarithm of the turns; cos and sin are
                             multiplied by `magnitude` (0.1 ln(factor) + 1 unless given)"""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError("rot_dim must be even and at least 2, got %r" % (rot_dim,))
    if n < 1:
        raise ValueError("the table needs at least one position")
    j = torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim
    kind, magnitude = (scaling[0] if scaling else None), 1.0
    if scaling and (len(scaling) < 2 or not scaling[1] > 0):
        raise ValueError("scaling needs a positive factor")
    if kind == "ntk":
        if rot_dim == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = base * scaling[1] ** (rot_dim / (rot_dim - 2))
    freq = base ** -j
    if kind == "linear":
        freq = freq / scaling[1]
    elif kind == "by_parts":
        if len(scaling) < 3:
            raise ValueError("by_parts scaling is (\"by_parts\", factor, trained, ...)")
        factor, trained = scaling[1:3]
        fast, slow = scaling[3:5] if len(scaling) > 3 else (32.0, 1.0)
        if not fast > slow > 0:
            raise ValueError("by_parts scaling needs fast > slow > 0")
        magnitude = scaling[5] if len(scaling) > 5 else 0.1 * math.log(factor) + 1.0
        turns = trained * freq / (2 * math.pi)
        stay = ((turns / slow).log() / math.log(fast / slow)).clamp(0, 1)
        freq = freq * stay + freq / factor * (1 - stay)
    elif kind not in (None, "ntk"):
        raise ValueError("unknown scaling %r: linear, ntk or by_parts" % (kind,))
    angle = torch.arange(n, dtype=torch.float64, device=device)[:, None] * freq
    return (torch.stack([angle.cos(), angle.sin()], -1) * magnitude).float()


def rotary(q, k, table, positions, *, interleaved=False, inverse=False):
    """Rotates q, and k with it unless it is None, by their positions: pair j of a head's first channels, (a, b) = channels
    (j, j + rot_dim/2), or (2j, 2j+1) where interleaved, becomes (a c - b s, b c + a s) with (c, s) = table[position, j]
    (rotary_table).  q [B,H,N,D] with positions [N] or [B,N], or packed [tokens, heads, D] with positions [tokens]; k likewise with
    heads of its own.  float16, bfloat16 or float32; computed in fp32 and rounded once.  inverse=True is the gradient of the call
    with inverse=False: the rotation back.  No autograd: where gradients are recorded, inputs that require them are refused; call it under
    torch.no_grad() or from the forward and backward of a torch.autograd.Function.  Returns q', or (q', k')."""
    return (_native_mod or _native()).rotary(q, k, table, positions, interleaved, inverse)


def append_int8_paged(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens=None, *, q=None, table=None,
                      interleaved=False):
    """Appends the new tokens' k and v [tokens, heads, D] (float16 or bfloat16) to a paged int8 cache, in place: k rotated by its
    position first where a `table` (rotary_table) is given, then both quantised with one scale for each block of tokens and head.
      k_cache, v_cache   int8 [pages, heads, page_size, D]: any page and head strides of 16 bytes, D 64, 128 or 256,
                         page_size a power of two from 8 to 256
      k_scale, v_scale   float32 [pages, heads, page_size/block], not negative; block 1 is one scale a token
      block_table        int32 [S, columns]: the page of a sequence's tokens i*page_size ...
      seq_lens           int32 [S]: tokens in the cache with the new ones, which are the last
      cu_seqlens         int32 [S+1]: where each sequence's new tokens begin among `tokens`; None: one token a sequence
    Where a block began in an earlier call its scale becomes the larger of the old one and the new tokens', and the codes of its older
    tokens follow.  Tokens behind the last sequence, and those of a sequence with seq_lens 0 (padding), are left out.  Two sequences may
    not append to one page in a call.  With q [tokens, query heads, D]: the same tokens' queries,
    rotated and quantised per token; returns (q8, q_scale [tokens, heads]) as attention_int8_paged takes them: zeros for a token whose position or page lies
    outside its table or cache (check_status() tells), not set for one that is left out."""
    return (_native_mod or _native()).append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens, q, table, interleaved)


def attention_int8_paged(q, k_cache, v_cache, q_scale, k_scale, v_scale, block_table, seq_lens, cu_seqlens, causal, sm_scale, *,
                         out_dtype=None, out=None, return_lse=False, debug_path=0):
    """Attention of packed int8 query rows q [tokens, query heads, D] over a paged int8 cache (append_int8_paged has the tensors):
    softmax(sm_scale * q k^T) v, with q = q8 * q_scale and the cache's values as codes times scales.  The rows of sequence s are
    cu_seqlens[s] .. cu_seqlens[s+1]-1 (None: one row each, decode); causal: they are its last tokens, row i of n sees keys up to
    seq_lens[s] - n + i, else all keys.  Sequences may share pages; keys whose page lies outside the cache do not count
    (check_status() tells).  Query heads share K/V heads in order, as in attention_int8.  A row that sees no key is
    zero.  Scores, softmax and sums are float32; p times the key's V scale is rounded to float16 (2^-11 of each, 2^-25 of the row's largest) for the
    product with the codes of v.  Returns o [tokens, query heads, D] in out_dtype (torch.float16 unless given, or torch.bfloat16); with `out` it is written there,
    and rows behind the last sequence stay as they were (without it they are not set).  return_lse: and the log2-domain LSE
    [tokens, query heads].  (debug_path: test hook, 1 or 2 for one of the two kernels whatever the sizes.)"""
    return (_native_mod or _native()).paged(q, k_cache, v_cache, q_scale, k_scale, v_scale, block_table, seq_lens, cu_seqlens, causal, sm_scale,
                                            out_dtype, out, return_lse, debug_path)
