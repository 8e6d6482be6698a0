"""Operator-level wrappers: same names, argument meaning and error behaviour as
the reference launch wrappers, over the C ABI.  No arithmetic happens here and no checks: the native host
path behind each of them (csrc/pyops.cpp) checks dtype, element count, contiguity and device of every tensor
against the problem sizes (the C ABI sees raw pointers and cannot), allocates the result the caller did not pass
and makes one library call on the current stream."""
import ctypes

import torch

from . import _lib

NF4 = 0
FP4 = 1
_native = _lib.native_ops()


def init():
    _lib.check(_lib.load().hq_init(), "hq_init")


def device_info():
    lib = _lib.load()
    v = [ctypes.c_int() for _ in range(5)]
    name = ctypes.create_string_buffer(256)
    _lib.check(lib.hq_device_info(*[ctypes.byref(x) for x in v], name, 256), "hq_device_info")
    return {"compute_units": v[0].value, "wavefront_size": v[1].value, "lds_bytes_per_cu": v[2].value,
            "memory_clock_khz": v[3].value, "memory_bus_bits": v[4].value, "name": name.value.decode()}


def q3_matvec(x, qweight, scales, zeros, out=None, accumulate=False):
    """y[n] = sum_k x[k]*(scales[n]*q[k][n] - zeros[n]); x fp32 or fp16 [K]."""
    return _native.q3_matvec(x, qweight, scales, zeros, out, accumulate)


def vecquant3matmul(vec, mat, mul, scales, zeros, height=None, width=None):
    """Reference signature (src/quant3MatMul-hip/kernels.h:171-190): mul += vec @ W."""
    # view(-1) never copies: a non-contiguous mul raises instead of losing the "mul +=" result in a temporary
    q3_matvec(vec.reshape(-1), mat, scales, zeros, out=_flat_inplace(mul, "mul"), accumulate=True)


def _flat_inplace(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor (it is updated in place)")
    return t.view(-1)


def vecquant3matmul_faster(vec, mat, mul, scales, zeros, height=None, width=None):
    """Reference signature (src/quant3MatMul-hip/kernels.h:193-217): fp16 vec, mul += vec @ W."""
    if vec.dtype != torch.float16:
        raise ValueError("vecquant3matmul_faster takes an fp16 vector")
    q3_matvec(vec.reshape(-1), mat, scales, zeros, out=_flat_inplace(mul, "mul"), accumulate=True)


def q3_gemm(A, qweight, scales, zeros, out=None):
    """out[m][n] = sum_k A[m][k]*(scales[n]*q[k][n] - zeros[n]); A fp16 [M][K]."""
    return _native.q3_gemm(A, qweight, scales, zeros, out)


def dequant_4bit(packed, absmax, n_elems, blocksize, table=NF4, out=None):
    return _native.dequant_4bit(packed, absmax, n_elems, blocksize, table, out)


def dynamic_map():
    """The signed dynamic 8-bit map of bitsandbytes (7 exponent bits), 256 sorted fp32 values in [-1, 1]: the
    table the reference ships as a literal (src/quantBnB-cuda/code.h).  Returns a CPU tensor."""
    import numpy as np
    f32 = np.float32
    vals = []
    for i in range(7):
        items = (1 << i) + 1
        step = (f32(1.0) - f32(0.1)) / f32(items - 1)
        b = [f32(0.1) + step * f32(j) if j < items // 2 else f32(1.0) - step * f32(items - 1 - j) for j in range(items)]
        sc = f32(10.0 ** (-6 + i))
        for j in range(items - 1):
            mean = (b[j] + b[j + 1]) / f32(2.0)
            vals += [sc * mean, -(sc * mean)]
    vals += [f32(0.0), f32(1.0)]
    return torch.from_numpy(np.sort(np.array(vals, dtype=f32)))


def quantize_dynamic8(code, A, out=None):
    return _native.quantize_dynamic8(code, A, out)


def lut_matmul(x, bW, alpha, q_bias, group_size, out=None):
    """matmul(output, input, nqW, m) of src/lut-gemm-hip/kernels.cu:27-31.
    bW uint32/int32 [K/32][nb][N], alpha fp16 [K/G][nb][N], q_bias fp16 [K/G][N] or None."""
    return _native.lut_matmul(x, bW, alpha, q_bias, group_size, out)


def code1x16_matvec(codes, x, codebooks, codebook_a_sizes, codebook_stride_int4, scales=None, out=None):
    """code1x16_matvec of src/quantAQLM-hip/main.cu:103-139 (plus the optional row scale)."""
    return _native.code1x16_matvec(codes, x, codebooks, codebook_a_sizes, codebook_stride_int4, scales, out)


def q3_pack(codes):
    """codes uint8 [K][N] (0..7) -> qweight int32 [3K/32][N]."""
    return _native.q3_pack(codes)


def bcq_pack(signs):
    """signs int8 [K][nb][N] (> 0 means +1) -> bW int32 [K/32][nb][N]."""
    return _native.bcq_pack(signs)


def quantize_4bit(x, blocksize, table=NF4):
    """x fp32/fp16 [n] -> (packed uint8 [ceil(n/2)], absmax fp32 [ceil(n/blocksize)])."""
    return _native.quantize_4bit(x, blocksize, table)


def static_scaled_int8_quant(x, scale, azp=None, out=None):
    """static_scaled_int8_quant of src/quantVLLM-hip/main.cu:133-148; x [tokens][hidden]."""
    return _native.int8_quant_static(x, float(scale), None if azp is None else int(azp), out)


def dynamic_scaled_int8_quant(x, with_azp=False, out=None):
    """dynamic_scaled_int8_quant of src/quantVLLM-hip/main.cu:150-168; returns (out, scales, azp or None)."""
    return _native.int8_quant_dynamic(x, with_azp, out)


def gemv_fp16(mat, vec, out=None):
    """solve_gemv_with_params of src/gemv-hip/gemv.cu:94-133: res = mat @ vec (fp16 in, fp32 sums, fp16 out)."""
    return _native.gemv_fp16(mat, vec, out)


def gemv_int8(mat, vec, scale, zero_point, out=None):
    """solve_gemv_int8_quantized_with_params of src/gemv-hip/gemv.cu:52-92 (mat int8 [rows][n])."""
    return _native.gemv_int8(mat, vec, float(scale), float(zero_point), out)


def gemv_int4(mat, vec, scale, zero_point, out=None):
    """solve_gemv_int4_quantized_with_params of src/gemv-hip/gemv.cu:10-50 (mat uint8 [rows][n/2], low nibble
    first)."""
    return _native.gemv_int4(mat, vec, float(scale), float(zero_point), out)


def mxfp4_qdq(x, out=None):
    """mxfp4<T>() of src/mxfp4-hip/main.cu:144-171: microscaling fp4 quantise-dequantise of an fp16 / bf16 tensor
    whose element count is a multiple of 32."""
    return _native.mxfp4_qdq(x, out)


def prompt_attention(q, k, v, cu_q, cu_k=None, causal=True, scale=None, out=None, window=None, sinks=0):
    """Attention over packed sequences: tokens cu_q[i] .. cu_q[i + 1] - 1 of q [tokens][heads][64 or 128] are sequence i's and see
    its keys cu_k[i] .. cu_k[i + 1] - 1 (cu_k: cu_q's) of k and v [keys][kv_heads][head size]; fp16 or bf16, int32 bounds.
    causal: the last token sees all keys, each one before it a key less; a token that sees none gets zeros.  scale: 1 / sqrt of the
    head size.  q, k and v may be parts of a fused projection's rows.  window, causal only: a token sees no more than the last `window`
    of its keys, its own among them, and the first `sinks` keys of its sequence.  Returns [tokens][heads][head size]; tokens of no sequence
    are left unwritten."""
    return _native.prompt_attention(q, k, v, cu_q, cu_k, causal, scale, out, window, sinks)


def paged_attention(q, k_pages, v_pages, table, lengths, groups=None, shared=None, scale=None, out=None):
    """Attention of one token per request over a paged cache: q [requests][heads][64 or 128] over the first lengths[s] tokens of
    row s, token t being token t % page of page table[s][t // page] in k_pages and v_pages [pages][kv_heads][page][head size].
    groups (int32 [n + 1]) and shared (int32 [n]): the first shared[g] tokens of the requests groups[g] .. groups[g + 1] - 1 are in the
    same pages, as cache_step leaves them, and are read once for all of them.  Tokens of a page: a power of two, 8 ... 1024."""
    return _native.paged_attention(q, k_pages, v_pages, table, lengths, groups, shared, scale, out)


def chunk_attention(q, k_pages, v_pages, table, lengths, cu_q, window=None, sinks=0, scale=None, out=None):
    """Attention of any number of new tokens per request - one, drafted ones, a chunk of a prompt - over a paged cache that holds their keys and
    values already: tokens cu_q[s] ... cu_q[s + 1] - 1 of q [tokens][heads][64 or 128] are the last of the first lengths[s] tokens of row s,
    token t being token t % page of page table[s][t // page] in k_pages and v_pages [pages][kv_heads][page][head size], and each sees the
    tokens up to itself.  window: no more than the last `window` of them, itself among them, and the first `sinks` tokens of its request;
    pages that no token sees are not read, and need not be there.  Returns [tokens][heads][head size]; a token that sees nothing gets
    zeros, tokens of no request are left unwritten.  Tokens of a page: a power of two, 8 ... 1024."""
    return _native.chunk_attention(q, k_pages, v_pages, table, lengths, cu_q, window, sinks, scale, out)


def cache_write(k, v, k_pages, v_pages, table, starts, cu):
    """Tokens cu[s] .. cu[s + 1] - 1 of k and v [tokens][kv_heads][head size] become tokens starts[s] and on of row s of the table;
    a token without a page is left out.  Tokens of a page: a power of two, 1 ... 1024."""
    _native.cache_write(k, v, k_pages, v_pages, table, starts, cu)


def cache_step(pool, page_size, table, lengths, refs, parent, add, out=None):
    """The page tables of the next step: row s goes on from row parent[s] of this one (-1: from nothing) and gets room for add[s]
    tokens more.  Whole pages are shared, a half-filled one is copied in every plane of pool [planes][pages][...] for each row but the
    first that goes on from it, new pages are the free ones (refs[p] <= 0), lowest first, to the rows in order.
    Returns (table, lengths, refs, starts, missing): starts are the lengths before the new tokens, missing (int32 [1]) the pages that
    there were not - a row ends where its pages end.  out: five tensors for them that share nothing with the arguments.
    page_size: any, but a cache that is to be written and attended to has a power of two, 8 ... 1024."""
    return _native.cache_step(pool, page_size, table, lengths, refs, parent, add, out)


def cache_compact(pool, table, refs, out=None):
    """Moves the pages in use (refs[p] > 0) behind the first n, n the number of pages in use, into the free ones among those, in order,
    in every plane of the pool.  Returns (table, refs, n as int32 [1])."""
    return _native.cache_compact(pool, table, refs, out)


def rotary_table(positions, rotary, base=10000.0, device="cuda"):
    """Cosines and sines of a head's angles at positions 0 ... positions - 1, as norm_rotate takes them: fp32 [positions][rotary], the
    cosines of position * base ** (-2 i / rotary), i < rotary / 2, and then their sines.  Angles in 64 bits: in 32, those of far positions
    are off by thousandths.  rotary: a multiple of 16."""
    if rotary < 0 or rotary % 16:
        raise ValueError(f"rotary must be a multiple of 16, got {rotary}")
    half = rotary // 2
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * float(base) ** (-torch.arange(half, dtype=torch.float64) / half)
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


def norm_rotate(q, k, cos_sin, positions, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, out=None):
    """Heads of queries and keys normed and rotated: each of q [tokens][heads][64 or 128] and k [tokens][kv_heads][head size], fp16 or bf16,
    becomes x * rsqrt(mean(x^2) + eps) * weight (weight [head size] of their type; None: is not normed; eps at least
    2 ** -126), and then its first cos_sin.size(1)
    elements (a multiple of 16) are rotated by row positions[t] of cos_sin, cosines and then sines of the angles (rotary_table; a position
    that is not in the table is cut to it): element i against element i + half of them, or, interleaved, 2 i against 2 i + 1.  cos_sin
    None: no rotation.  fp32, one rounding.  q and k may be parts of a fused projection's rows.  Returns (q, k), new tensors or
    out's two, which may be parts of rows as well, q and k themselves among them."""
    q_out, k_out = (None, None) if out is None else out
    return _native.norm_rotate(q, k, cos_sin, positions, q_weight, k_weight, eps, interleaved, q_out, k_out)


def cache_write_rotated(q, k, v, k_pages, v_pages, table, starts, cu, cos_sin, q_weight=None, k_weight=None, eps=1e-6, interleaved=False,
                        out=None):
    """norm_rotate and cache_write in one: tokens cu[s] ... cu[s + 1] - 1 become tokens starts[s] and on of row s of the table, which is
    their position too; the keys, normed and rotated, and the values go into the pages, as cache_write would take them.  Returns the
    queries, normed and rotated (out: parts of rows, q itself among them); those of tokens of no row are left unwritten."""
    return _native.cache_write_rotated(q, k, v, k_pages, v_pages, table, starts, cu, cos_sin, q_weight, k_weight, eps, interleaved, out)
