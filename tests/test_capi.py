"""The C-ABI library without a GPU: it loads, exports every declared symbol,
and rejects bad arguments with the documented codes before launching
anything (validation runs before any HIP call)."""
import ctypes

import pytest

from teenyformers_amd import _lib

OK, NULLP, SHAPE, UNSUP, WS, VALUE, SCRATCH, NOT_INIT = 0, -1, -2, -3, -4, -7, -8, -9
GRAD_F32 = 0x100
F32, BF16 = 0, 1
NEG_INF = float("-inf")
P = 0x1000  # a non-null dummy pointer: never dereferenced by failing calls


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def test_exports_every_declared_symbol(L):
    declared = _lib.header_functions()
    assert len(declared) >= 20
    for name in declared:
        assert hasattr(L, name), name
    assert L.teeny_abi_version() == 1


def test_strerror(L):
    assert L.teeny_strerror(0).decode() == "ok"
    assert "workspace" in L.teeny_strerror(WS).decode()


def fwd(L, **kw):
    a = dict(q=P, k=P, v=P, o=P, l=P, nq=128, nk=128, scale=0.125, neg_inf=NEG_INF, b=1, hq=4,
             hkv=4, d=64, dtype=BF16)
    a.update(kw)
    return L.teeny_causal_flash_attn2_fwd(a["q"], a["k"], a["v"], a["o"], a["l"], a["nq"], a["nk"],
                                          a["scale"], a["neg_inf"], a["b"], a["hq"], a["hkv"],
                                          a["d"], a["dtype"], None)


def test_fa2_fwd_validation(L):
    assert fwd(L, q=None) == NULLP
    assert fwd(L, l=None) == NULLP
    assert fwd(L, nq=0) == SHAPE
    assert fwd(L, hq=6, hkv=4) == SHAPE  # Hq must be a multiple of Hkv
    assert fwd(L, d=96) == UNSUP
    assert fwd(L, d=32, dtype=BF16) == UNSUP  # bf16 built for 64/128
    assert fwd(L, dtype=7) == UNSUP
    assert fwd(L, neg_inf=-1e9) == VALUE  # the reference always passes -inf
    assert fwd(L, scale=float("nan")) == VALUE


def test_fa2_fwd_merged_validation(L):
    """The merged-heads forward validates like the forward and is bf16 only."""
    def m(causal=1, **kw):
        a = dict(q=P, nq=128, scale=0.125, dtype=BF16)
        a.update(kw)
        return L.teeny_flash_attn2_fwd_merged(a["q"], P, P, P, P, a["nq"], 128, a["scale"],
                                              NEG_INF, 1, 4, 4, 64, a["dtype"], causal, None)
    for c in (0, 1):
        assert m(c, dtype=F32) == UNSUP
        assert m(c, q=None) == NULLP
        assert m(c, nq=0) == SHAPE
        assert m(c, scale=0.0) == VALUE


def test_fa2_fwd_qkv_and_rope_table_validation(L):
    """The attention from the fused QKV projection validates like the
    forward, is bf16 only and needs a 16-byte aligned (cos, sin) table."""
    def f(**kw):
        a = dict(qkv=P, cs=P, nq=128, dtype=BF16, scale=0.125, d=64)
        a.update(kw)
        return L.teeny_flash_attn2_fwd_qkv(a["qkv"], a["cs"], P, P, P, P, a["nq"], 128, a["scale"],
                                           NEG_INF, 1, 4, 2, a["d"], a["dtype"], 1, None)
    assert f(dtype=F32) == UNSUP
    assert f(cs=None) == NULLP
    assert f(cs=P + 8) == VALUE
    assert f(qkv=None) == NULLP
    assert f(nq=0) == SHAPE
    assert f(d=96) == UNSUP
    assert f(scale=0.0) == VALUE
    assert f(nq=1 << 22, d=128) == SHAPE  # B*S*(Hq+2Hkv)*D past the 32-bit element range
    assert L.teeny_rope_table(None, 16, 64, 9.2, None) == NULLP
    assert L.teeny_rope_table(P, 0, 64, 9.2, None) == SHAPE
    assert L.teeny_rope_table(P, 16, 64, 9.2, None) == SHAPE  # positions in blocks of 32
    assert L.teeny_rope_table(P, 32, 40, 9.2, None) == SHAPE  # head_dim a multiple of 16
    assert L.teeny_rope_table(P, 32, 64, float("inf"), None) == VALUE


def test_fa2_scale_domain(L):
    """bf16 kernels fold the scale into the exponent after masking raw
    scores to -inf: scale must be > 0 there (0 or negative would turn masked
    scores into NaN or +inf)."""
    assert fwd(L, scale=0.0) == VALUE
    assert fwd(L, scale=-0.125) == VALUE
    assert fwd(L, scale=float("inf")) == VALUE
    ws = L.teeny_flash_attn2_bwd_workspace_bytes(128, 1, 4, 64, BF16)
    rc = L.teeny_causal_flash_attn2_bwd(P, P, P, P, P, P, P, P, P, 128, 128, 0.0, 1, 4, 4, 64,
                                        BF16, P, ws, None)
    assert rc == VALUE
    rc = L.teeny_decode_attention(P, P, P, P, 1, 4, 4, 10, 16, 64, -1.0, BF16, P, 1 << 20, None)
    assert rc == VALUE


def test_fa2_grad_f32_flag(L):
    """TEENY_GRAD_F32 changes the gradients' type, not the workspace."""
    for args in ((4096, 8, 32, 128), (300, 2, 8, 128), (128, 1, 4, 64)):
        assert L.teeny_flash_attn2_bwd_workspace_bytes(*args, BF16 | GRAD_F32) == \
            L.teeny_flash_attn2_bwd_workspace_bytes(*args, BF16)
    f = L.teeny_flash_attn2_bwd_workspace_bytes_gqa
    assert f(16384, 16384, 1, 64, 8, 128, BF16 | GRAD_F32) == \
        f(16384, 16384, 1, 64, 8, 128, BF16)
    # validation still applies to the flagged dtype
    rc = L.teeny_causal_flash_attn2_bwd(P, P, P, P, P, P, P, P, P, 128, 128, 0.125, 1, 4, 4, 32,
                                        BF16 | GRAD_F32, P, 1 << 20, None)
    assert rc == UNSUP


def test_noalloc_bwd_refuses_beyond_scratch(L):
    """The no-allocation backward's static array is 16 MiB per device;
    problems whose workspace exceeds it are refused before anything runs."""
    assert L.teeny_scratch_bytes() == 16 << 20
    # B8 Hq32 S4096 D128 needs 8 MiB: within; B8 Hq32 S16384 needs 32 MiB
    assert L.teeny_flash_attn2_bwd_workspace_bytes(4096, 8, 32, 128, BF16) <= 16 << 20
    assert L.teeny_flash_attn2_bwd_workspace_bytes(16384, 8, 32, 128, BF16) > 16 << 20
    rc = L.teeny_causal_flash_attn2_bwd_noalloc(P, P, P, P, P, P, P, P, P, 16384, 16384, 0.088,
                                                8, 32, 32, 128, BF16, None)
    assert rc == SCRATCH
    assert "scratch" in L.teeny_strerror(SCRATCH).decode()


def test_fa2_bwd_workspace_gqa(L):
    """The larger workspace that allows the dK/dV head split: only for bf16
    GQA with an even group, 12288+ query rows and few key blocks (at most
    four 128-key blocks x batch x kv heads per CU of a 256-CU device without
    a GPU to ask): fp32 dK and dV partials for 4 splits (2 when 4 does not
    divide the group) on top of the base workspace."""
    f = L.teeny_flash_attn2_bwd_workspace_bytes_gqa
    base = L.teeny_flash_attn2_bwd_workspace_bytes
    # B1 Hq64 Hkv8 S16384: 128 blocks x 8 kv heads = 1024 workgroups, split 4
    assert f(16384, 16384, 1, 64, 8, 128, BF16) == base(16384, 1, 64, 128, BF16) + \
        2 * 4 * 8 * 16384 * 128 * 4
    # group of 2: split 2 (the shape the no-allocation test runs)
    assert f(12288, 12288, 1, 2, 1, 64, BF16) == base(12288, 1, 2, 64, BF16) + \
        2 * 2 * 1 * 12288 * 64 * 4
    # 2048-12287 rows (two wavefront groups, no partials), short walks, MHA,
    # odd groups, many key blocks, fp32: nothing to split
    for args in ((8191, 8191, 1, 64, 8, 128), (4096, 4096, 2, 32, 8, 128),
                 (1024, 1024, 4, 32, 8, 128), (512, 512, 16, 32, 8, 128),
                 (16384, 16384, 1, 32, 32, 128), (16384, 16384, 1, 24, 8, 128),
                 (16384, 16384, 2, 64, 8, 128)):
        Sq, Sk, B, Hq, Hkv, D = args
        assert f(*args, BF16) == base(Sq, B, Hq, D, BF16), args
    assert f(128, 128, 1, 4, 2, 64, F32) == base(128, 1, 4, 64, F32)
    assert f(16384, 16384, 1, 64, 8, 128, F32) == base(16384, 1, 64, 128, F32)
    assert f(128, 128, 1, 6, 4, 64, BF16) == 0  # Hq % Hkv != 0
    assert f(0, 128, 1, 4, 2, 64, BF16) == 0


def test_fa2_bwd_workspace(L):
    need = L.teeny_flash_attn2_bwd_workspace_bytes(4096, 8, 32, 128, BF16)
    rows = 8 * 32 * 4096
    assert need >= rows * 4  # Delta
    assert L.teeny_flash_attn2_bwd_workspace_bytes(128, 1, 4, 64, F32) >= 4 * 128 * 4
    small = L.teeny_flash_attn2_bwd_workspace_bytes(128, 1, 4, 64, BF16)
    rc = L.teeny_causal_flash_attn2_bwd(P, P, P, P, P, P, P, P, P, 128, 128, 0.125, 1, 4, 4, 64,
                                        BF16, P, small - 1, None)
    assert rc == WS
    rc = L.teeny_causal_flash_attn2_bwd(P, P, P, P, P, P, P, P, P, 128, 128, 0.125, 1, 4, 4, 64,
                                        BF16, None, 1 << 30, None)
    assert rc == WS


def test_other_ops_validation(L):
    assert L.teeny_rope_fwd(P, P, 8, 9.21, 2, 12, BF16, None) == UNSUP  # 12 % 8
    assert L.teeny_rope_fwd(None, P, 8, 9.21, 2, 16, F32, None) == NULLP
    assert L.teeny_rope_fwd(P, P, 8, 9.21, 2, 24, F32, None) == UNSUP  # not a power of two
    assert L.teeny_transpose_heads(P, P, 0, 4, 1, 64, BF16, None) == SHAPE
    assert L.teeny_transpose_heads(P, P, 8, 4, 1, 64, BF16, None) == VALUE  # src == dst
    assert L.teeny_rmsnorm_fwd(P, P, None, P, 4, 64 * 8 * 32, 1e-5, BF16, None) == UNSUP
    assert L.teeny_fused_add_rmsnorm_fwd(P, P, P, P, None, P, 4, 16, 1e-6, F32, None) == NULLP
    assert L.teeny_fused_add_rmsnorm_bwd(P, P, P, P, P, P, P, 4, 16, F32, None, 0, None) == WS
    assert L.teeny_rmsnorm_bwd_set(0, P, P, P, P, P, P, P, 4, 16, F32, P, 1 << 20, None) == VALUE
    assert L.teeny_rmsnorm_bwd_set(1, P, P, P, P, P, P, P, 4, 16, F32, None, 0, None) == WS
    assert L.teeny_swiglu_fwd(P, P, 0, 8, F32, None) == SHAPE
    assert L.teeny_token_embed_fwd(P, P, P, 4, 16, 10, BF16, F32, None) == UNSUP  # ids dtype


def test_add_validation(L):
    assert L.teeny_add(None, P, P, 16, BF16, None) == NULLP
    assert L.teeny_add(P, P, P, 0, BF16, None) == SHAPE
    assert L.teeny_add(P + 2, P, P, 16, BF16, None) == VALUE  # not 16-byte aligned
    assert L.teeny_add(P, P, P, 16, 9, None) == UNSUP


def test_decode_ops_validation(L):
    # linear: any M; the matrix-core GEMM needs N % 64 and K % 64 (the
    # decode-step kernels, M <= 16, N % 128 and K % 128)
    assert L.teeny_linear_bf16(P, P, P, 17, 96, 128, None) == UNSUP
    assert L.teeny_linear_bf16(P, P, P, 16, 64, 96, None) == UNSUP
    assert L.teeny_linear_bf16(P, P, P, 300, 128, 4100, None) == UNSUP
    assert L.teeny_linear_bf16(P, P, P, 300, 128, 1 << 22, None) == SHAPE  # 32-bit offsets
    # linear_swiglu: the GEMM needs F % 32 and K % 64 (the decode kernel,
    # M <= 16, F % 64 and K % 128)
    assert L.teeny_linear_swiglu_bf16(P, P, P, 17, 48, 128, None) == UNSUP
    assert L.teeny_linear_swiglu_bf16(P, P, P, 300, 64, 96, None) == UNSUP
    assert L.teeny_linear_swiglu_bf16(P, P, P, 300, 64, 1 << 22, None) == SHAPE
    # the same K limit where 17 to 64 rows stream the weight
    assert L.teeny_linear_swiglu_bf16(P, P, P, 64, 64, 1 << 22, None) == SHAPE
    for m in (4, 64, 300):
        assert L.teeny_gemm_bf16(P, P, P, m, 128, 1 << 22, None) == SHAPE
    assert L.teeny_linear_swiglu_bf16(P, None, P, 300, 64, 128, None) == NULLP
    assert L.teeny_linear_bf16(None, P, P, 16, 128, 128, None) == NULLP
    assert L.teeny_linear_bf16(P, P, P, 0, 128, 128, None) == SHAPE
    assert L.teeny_linear_swiglu_bf16(P, P, P, 4, 48, 128, None) == UNSUP
    assert L.teeny_linear_partials_bf16(P, P, P, 4, 128, 4096, 1000, None) == VALUE
    assert L.teeny_linear_partials_bf16(P, P, P, 4, 128, 4096, 0, None) == VALUE
    assert L.teeny_linear_partials_count(4096, 1024) == 4
    assert L.teeny_linear_partials_count(14336, 2048) == 7
    assert L.teeny_linear_partials_count(4096, 8192) == 1
    assert L.teeny_fused_add_rmsnorm_partials_fwd(P, 0, P, P, P, P, P, 4, 1024, 1e-5, BF16,
                                                  None) == SHAPE
    assert L.teeny_fused_add_rmsnorm_partials_fwd(None, 2, P, P, P, P, P, 4, 1024, 1e-5, BF16,
                                                  None) == NULLP
    assert L.teeny_qkv_rope_split_partials_dev(P, 2, P, P, P, 4, 1, None, 64, 8, 2, 64,
                                               9.21, BF16, None) == NULLP
    assert L.teeny_qkv_rope_split_partials_dev(P, 2, P, P, P, 4, 1, P, 64, 8, 3, 64,
                                               9.21, BF16, None) == SHAPE  # 8 % 3
    assert L.teeny_argmax_rows(None, P, 4, 10, BF16, None) == NULLP
    assert L.teeny_argmax_rows(P, P, 0, 10, BF16, None) == SHAPE
    assert L.teeny_argmax_rows_advance(None, P, 4, 10, BF16, P, None) == NULLP
    assert L.teeny_embed_rmsnorm_fwd(P, P, P, P, P, 256, 64, 10, 1e-5, 3, BF16, None) == UNSUP
    assert L.teeny_embed_rmsnorm_fwd(P, P, P, P, P, 4, 60, 10, 1e-5, 3, BF16, None) == UNSUP
    assert L.teeny_embed_rmsnorm_fwd(P, P, P, P, P, 4, 64, 10, 1e-5, F32, BF16, None) == UNSUP
    assert L.teeny_embed_rmsnorm_fwd(P, P, P, P, None, 4, 64, 10, 1e-5, 3, BF16, None) == NULLP


def test_decode_qkv_attention_validation(L):
    def call(**kw):
        a = dict(parts=P, n=4, k=P, v=P, o=P, b=2, hq=32, hkv=8, d=128, cl=640, pos=P,
                 lnb=13.1, scale=0.088, dtype=BF16)
        a.update(kw)
        return L.teeny_decode_qkv_attention_dev(a["parts"], a["n"], a["k"], a["v"], a["o"], a["b"],
                                                a["hq"], a["hkv"], a["d"], a["cl"], a["pos"],
                                                a["lnb"], a["scale"], a["dtype"], None)
    assert call(parts=None) == NULLP
    assert call(pos=None) == NULLP
    assert call(dtype=F32) == UNSUP
    assert call(d=96) == UNSUP
    assert call(hq=64, hkv=1) == UNSUP  # 64 q heads per kv head: more than one product's rows
    assert call(hq=6, hkv=4) == SHAPE
    assert call(n=0) == SHAPE
    assert call(scale=-1.0) == VALUE
    assert call(lnb=float("nan")) == VALUE


def test_fa2_32bit_row_offsets(L):
    """bf16 kernels address a head's rows through 32-bit buffer offsets: a
    head of n_ctx * D * 2 >= 2^31 bytes (Q or dO of 8.4M rows at D = 128,
    fewer than 2^31 elements in all) is refused before any launch, on the
    query side as on the key side."""
    big = 8_400_000  # 8.4M * 128 * 2 B = 2.15e9 B; 8.4M * 128 = 1.08e9 elements
    assert fwd(L, nq=big, nk=128, hq=1, hkv=1, d=128) == SHAPE
    assert fwd(L, nq=128, nk=big, hq=1, hkv=1, d=128) == SHAPE
    ws = 1 << 30
    for nq, nk in ((big, 128), (128, big)):
        rc = L.teeny_causal_flash_attn2_bwd(P, P, P, P, P, P, P, P, P, nq, nk, 0.088, 1, 1, 1,
                                            128, BF16, P, ws, None)
        assert rc == SHAPE, (nq, nk)
    # fp32 kernels index elements, not byte ranges: the element bound applies
    assert fwd(L, nq=big, nk=128, hq=1, hkv=1, d=128, dtype=F32) != SHAPE


def test_decode_qkv_attention_splits(L):
    """Key splits of the fused decode attention on a 256-CU device (here,
    without a GPU to ask): at most 16 workgroups per (b, kv head), and only
    for the keys attended that pay the merge."""
    at = L.teeny_decode_qkv_attention_splits_at
    assert [at(1, 8, 128, 4096, n) for n in (1, 1024, 1025, 4096, 9999)] == [1, 1, 16, 16, 16]
    assert [at(b, 8, 128, 4096, 4096) for b in (2, 4, 8, 10, 11, 16, 64)] == [16, 8, 4, 3, 2, 1, 1]
    assert [at(15, 8, 128, 4096, n) for n in (2048, 2049)] == [1, 2]  # two shares: twice the keys
    assert at(1, 8, 128, 1100, 1100) == 5  # a key tile per wavefront
    # heads of 64: half the bytes, from 33 (b, kv head) pairs on twice the keys
    assert [at(16, 2, 64, 4096, n) for n in (1024, 1025)] == [1, 8]
    assert [at(33, 1, 64, 4096, n) for n in (2048, 2049)] == [1, 7]
    assert [at(31, 4, 64, 8192, n) for n in (4096, 4097)] == [1, 2]
    assert at(0, 8, 128, 4096, 1) == at(1, 8, 128, 4096, 0) == 0
    assert [L.teeny_decode_qkv_attention_splits(1, 8, n) for n in (1024, 4096)] == [1, 16]
    assert L.teeny_decode_qkv_attention_splits(11, 8, 1100) == 1


def test_decode_qkv_attention_32bit_cache_offsets(L):
    """One (b, kv head) cache slab of cache_len * D * 2 >= 2^31 bytes is refused."""
    rc = L.teeny_decode_qkv_attention_dev(P, 1, P, P, P, 1, 1, 1, 128, 8_400_000, P, 13.1,
                                          0.088, BF16, None)
    assert rc == SHAPE
    rc = L.teeny_decode_qkv_attention_dev(P, 1, P, P, P, 1, 1, 1, 128, 4_000_000, P, 13.1,
                                          0.088, BF16, None)
    assert rc != SHAPE  # within range: fails later (no GPU here), not on the shape


def test_noalloc_needs_init(L):
    """The no-allocation backward loads and looks up nothing itself: without
    a device (here) it reports the HIP error, never a launch; its
    not-initialised code has its own text."""
    rc = L.teeny_causal_flash_attn2_bwd_noalloc(P, P, P, P, P, P, P, P, P, 128, 128, 0.125, 1,
                                                4, 4, 64, BF16, None)
    assert rc in (-5, NOT_INIT)
    assert "teeny_init" in L.teeny_strerror(NOT_INIT).decode()


def test_linear_f32_validation(L):
    """fp32 Linear (teeny_linear_f32 / teeny_gemm_f32): any M and N, K a
    multiple of 4, 16-byte aligned operands."""
    for fn in (L.teeny_linear_f32, L.teeny_gemm_f32):
        assert fn(None, P, P, 4, 8, 8, None) == NULLP
        assert fn(P, P, P, 0, 8, 8, None) == SHAPE
        assert fn(P, P, P, 4, 8, 6, None) == UNSUP
        assert fn(P + 4, P, P, 4, 8, 8, None) == VALUE
        assert fn(P, P + 8, P, 4, 8, 8, None) == VALUE


def test_stream_layout_validation(L):
    """The streaming layout (N % 16, K % 128, no overlap) and the linears
    that read it (the decode kernels' shapes only: M <= 16, N % 128 or
    F % 64, K % 128)."""
    Q = P + (1 << 30)  # a second buffer far from P
    assert L.teeny_linear_stream_layout_bf16(None, Q, 16, 128, None) == NULLP
    assert L.teeny_linear_stream_layout_bf16(P, Q, 0, 128, None) == SHAPE
    assert L.teeny_linear_stream_layout_bf16(P, Q, 24, 128, None) == UNSUP
    assert L.teeny_linear_stream_layout_bf16(P, Q, 16, 96, None) == UNSUP
    assert L.teeny_linear_stream_layout_bf16(P, P, 16, 128, None) == VALUE  # in place
    assert L.teeny_linear_stream_layout_bf16(P, P + 2 * 16 * 128 - 2, 16, 128, None) == VALUE
    assert L.teeny_linear_stream_layout_bf16(P, Q, 1 << 16, 1 << 16, None) == SHAPE
    assert L.teeny_linear_sl_bf16(None, P, P, 4, 128, 128, None) == NULLP
    assert L.teeny_linear_sl_bf16(P, P, P, 17, 128, 128, None) == UNSUP  # prompt sizes: row-major
    assert L.teeny_linear_sl_bf16(P, P, P, 4, 96, 128, None) == UNSUP
    assert L.teeny_linear_sl_bf16(P, P, P, 4, 128, 192, None) == UNSUP
    assert L.teeny_linear_swiglu_sl_bf16(P, P, P, 4, 96, 128, None) == UNSUP
    assert L.teeny_linear_swiglu_sl_bf16(P, P, P, 0, 64, 128, None) == SHAPE
    assert L.teeny_linear_partials_sl_bf16(P, P, P, 4, 128, 4096, 1000, None) == VALUE
    assert L.teeny_linear_partials_sl_bf16(P, P, P, 4, 128, 4096, 0, None) == VALUE
    assert L.teeny_linear_partials_sl_bf16(P, None, P, 4, 128, 4096, 512, None) == NULLP


def test_header_is_c(tmp_path):
    """include/teeny_hip.h is a C header: a C99 program that includes it
    compiles without warnings, links against libteeny_hip.so and calls it
    (what a cgo / bindgen / ctypes consumer relies on)."""
    import os
    import shutil
    import subprocess

    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    libdir = os.path.join(root, "teenyformers_amd")
    src = tmp_path / "use_header.c"
    src.write_text('#include "teeny_hip.h"\n'
                   "int main(void) { return teeny_abi_version() == 1 ? 0 : 1; }\n")
    exe = tmp_path / "use_header"
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.run([gcc, "-std=c99", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__",
                    "-I" + os.path.join(root, "include"), "-I" + os.path.join(rocm, "include"),
                    str(src), "-L" + libdir, "-lteeny_hip", "-Wl,-rpath," + libdir,
                    "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)]).returncode == 0


def test_rope_base_tensor_by_value():
    """The kept ln(base) follows the value of a base given as a tensor."""
    import torch

    from teenyformers_amd import ops
    base = torch.tensor(1e4)
    first = ops._ln(base)
    base.fill_(5e5)
    assert first == ops._ln(1e4) and ops._ln(base) == ops._ln(5e5) != first


def test_fused_decode_cache_limit(monkeypatch):
    """A one-token step over a cache slab that the fused decode attention does
    not address (2 GiB of one kv head) takes the unfused path, however many
    workgroups would share its keys."""
    from types import SimpleNamespace

    import torch

    from teenyformers_amd import llama, ops
    cfg = llama.LlamaConfig(d_model=512, n_heads=4, n_kv_heads_=1)
    model = llama.Llama(cfg, {})
    qkv = ops.Partials(torch.empty(1, 1, 768), (1, 1, 768), torch.bfloat16)
    monkeypatch.setattr(ops, "decode_qkv_splits", lambda *a: 16)
    assert model._fused_decode(qkv, SimpleNamespace(capacity=8_388_607))
    assert not model._fused_decode(qkv, SimpleNamespace(capacity=8_388_608))


def test_sample_rows_validation(L):
    """The sampler's refusals, and the workspace sizes of shapes that it does not take."""
    def f(**kw):
        a = dict(x=P, ld=100, u=P, rows=4, cols=100, t=1.0, ts=None, k=0, ks=None, p=1.0, ps=None, m=0.0,
                 ms=None, out=P, dtype=BF16, adv=None, ws=P, wsb=1 << 40)
        a.update(kw)
        return L.teeny_sample_rows(a["x"], a["ld"], a["u"], a["rows"], a["cols"], a["t"], a["ts"], a["k"],
                                   a["ks"], a["p"], a["ps"], a["m"], a["ms"], a["out"], a["dtype"],
                                   a["adv"], a["ws"], a["wsb"], None)
    nan = float("nan")
    for kw in (dict(x=None), dict(u=None), dict(out=None)):
        assert f(**kw) == NULLP
    assert f(dtype=7) == UNSUP
    for kw in (dict(rows=0), dict(rows=65536), dict(cols=0), dict(cols=524281), dict(ld=99),
               dict(ld=-100)):
        assert f(**kw) == SHAPE
    for kw in (dict(t=-1.0), dict(t=nan), dict(k=-1), dict(p=0.0), dict(p=1.01), dict(p=nan), dict(m=-0.1),
               dict(m=1.1), dict(m=nan), dict(x=P + 1), dict(ws=P + 8)):
        assert f(**kw) == VALUE
    need = L.teeny_sample_rows_workspace_bytes(4, 100)
    assert need > 0 and f(wsb=need - 1) == WS and f(ws=None) == WS
    for rows, cols in ((0, 5), (65536, 5), (5, 0), (5, 524281)):
        assert L.teeny_sample_rows_workspace_bytes(rows, cols) == 0


def test_shared_prefix_attention_validation(L):
    """Refusals of the attention over a shared prefix."""
    def f(**kw):
        a = dict(q=P, kp=P, vp=P, k=P, v=P, o=P, b=2, hq=4, hkv=2, s=1, np=100, lp=128, past=None, st=0,
                 host=5, L=64, d=64, scale=0.125, merged=0, dtype=BF16, ws=P, wsb=1 << 40)
        a.update(kw)
        return L.teeny_shared_prefix_attention(
            a["q"], a["kp"], a["vp"], a["k"], a["v"], a["o"], a["b"], a["hq"], a["hkv"], a["s"], a["np"],
            a["lp"], a["past"], a["st"], a["host"], a["L"], a["d"], a["scale"], a["merged"], a["dtype"],
            a["ws"], a["wsb"], None)
    for n in ("q", "kp", "vp", "k", "v", "o"):
        assert f(**{n: None}) == NULLP
    for kw in (dict(d=96), dict(d=32), dict(dtype=7), dict(d=256, dtype=F32)):
        assert f(**kw) == UNSUP
    for kw in (dict(b=0), dict(hq=3), dict(hkv=0), dict(s=0), dict(np=-1), dict(np=129), dict(L=0),
               dict(s=65), dict(L=1 << 24), dict(lp=1 << 24), dict(b=1 << 25)):
        assert f(**kw) == SHAPE, kw
    for kw in (dict(host=-1), dict(host=64), dict(past=P, st=2), dict(scale=0.0), dict(q=P + 2),
               dict(o=P + 8), dict(kp=P + 4), dict(scale=float("inf"))):
        assert f(**kw) == VALUE, kw
    assert f(q=P + 2, dtype=F32) == VALUE
    # (few keys need none)
    assert L.teeny_shared_prefix_attention_workspace_bytes(2, 4, 2, 1, 100, 64, 64, BF16) == 0
    need = L.teeny_shared_prefix_attention_workspace_bytes(2, 4, 2, 1, 100, 3000, 64, BF16)
    assert need > 0 and f(L=3000, wsb=need - 1) == WS and f(L=3000, ws=None) == WS
    assert f(L=3000, ws=P + 8) == VALUE
    assert L.teeny_shared_prefix_attention_workspace_bytes(2, 4, 2, 1, 100, 64, 64, F32) > 0
    assert L.teeny_shared_prefix_attention_workspace_bytes(2, 4, 2, 1, 30, 64, 64, F32) == 0
    assert L.teeny_shared_prefix_attention_workspace_bytes(2, 3, 2, 1, 100, 64, 64, BF16) == 0
    assert L.teeny_shared_prefix_attention_workspace_bytes(2, 4, 2, 1, -1, 64, 64, BF16) == 0


def test_qkv_rope_split_rows_validation(L):
    """Refusals of the QKV split behind a prefix."""
    def f(**kw):
        a = dict(qkv=P, parts=None, n=0, q=P, k=P, v=P, b=2, s=1, row0=None, st=0, host=3, off=10, L=64,
                 hq=4, hkv=2, d=64, ln=9.2, dtype=BF16)
        a.update(kw)
        return L.teeny_qkv_rope_split_rows(a["qkv"], a["parts"], a["n"], a["q"], a["k"], a["v"], a["b"],
                                           a["s"], a["row0"], a["st"], a["host"], a["off"], a["L"],
                                           a["hq"], a["hkv"], a["d"], a["ln"], a["dtype"], None)
    for kw in (dict(qkv=None), dict(parts=P, n=1), dict(q=None), dict(k=None), dict(v=None)):
        assert f(**kw) == NULLP, kw
    for kw in (dict(host=-1), dict(host=64), dict(s=0), dict(hq=5), dict(qkv=None, parts=P, n=0)):
        assert f(**kw) == SHAPE, kw
    for kw in (dict(off=-1), dict(off=(1 << 30) + 1), dict(row0=P, st=2), dict(ln=float("nan"))):
        assert f(**kw) == VALUE, kw
    assert f(dtype=7) == UNSUP and f(d=12) == UNSUP


def test_generate_command_refuses(capsys):
    """Arguments out of their ranges end the command before anything is loaded."""
    from teenyformers_amd import generate
    for bad in (["--num-samples", "0"], ["--top-k", "-1"], ["--top-p", "0"], ["--top-p", "1.5"],
                ["--min-p", "-0.1"], ["--min-p", "2"], ["--temperature", "-1"], ["--temperature", "nan"]):
        with pytest.raises(SystemExit):
            generate.main(["--preset", "llama3-8b", *bad])


def test_qkv_split_behind_a_prefix_needs_q():
    """ops.qkv_rope_split without q_out is the prompt's form: refused by name elsewhere."""
    import torch

    from teenyformers_amd import ops
    qkv, cache = torch.zeros(2, 1, 512), torch.zeros(2, 2, 4, 64)
    for kw in (dict(pos0=0, rope_offset=5), dict(pos0=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="q_out is required"):
            ops.qkv_rope_split(qkv, None, cache, cache, n_heads_q=4, n_heads_kv=2, rope_base=1e4, **kw)
    # (a tensor elsewhere than on a GPU is refused as before)
    with pytest.raises(ValueError, match="device"):
        ops.qkv_rope_split(qkv, torch.zeros(2, 4, 1, 64), cache, cache, 0, 4, 2, 1e4, rope_offset=5)


def test_shared_prefix_of_two_shapes():
    """A prefix's K and V are one cache's: V of two sequences is refused, not cut."""
    import torch

    from teenyformers_amd import ops
    q, c = torch.zeros(2, 4, 64), torch.zeros(2, 2, 8, 64)
    k, v = torch.zeros(1, 2, 5, 64), torch.zeros(2, 2, 5, 64)
    for a, b in ((k, v), (v, k), (k, k[0]), (k[0], k), (k, k[:, :, :4])):
        with pytest.raises(ValueError, match="of one shape"):
            ops.shared_prefix_attention(q, a, b, c, c, 5, 0)


def test_paged_validation(L):
    def split(**kw):
        a = dict(qkv=P, parts=None, n_parts=0, q=P, k=P, v=P, table=P, ld=8, width=8, starts=None, past=P,
                 host=0, b=2, t=2, n_pages=9, page=16, hq=8, hkv=2, d=128, ln=9.2, dtype=BF16)
        a.update(kw)
        return L.teeny_paged_qkv_rope_split(*a.values(), None)

    def att(**kw):
        a = dict(q=P, k=P, v=P, o=P, table=P, ld=8, width=8, starts=None, past=P, host=0, b=2, t=2, new=1,
                 keys=128, n_pages=9, page=16, hq=8, hkv=2, d=128, scale=0.1, dtype=BF16, ws=P, size=1 << 30)
        a.update(kw)
        return L.teeny_paged_attention(*a.values(), None)

    for f in (split, att):
        for name in ("q", "k", "v", "table"):
            assert f(**{name: None}) == NULLP, name
        for kw in (dict(b=0), dict(t=-1), dict(t=3), dict(width=0), dict(ld=7), dict(n_pages=0), dict(page=8),
                   dict(page=24), dict(page=2048), dict(hkv=3), dict(hq=0), dict(t=1 << 24),
                   dict(width=1 << 27, ld=1 << 27)):
            assert f(**kw) == SHAPE, kw
        assert f(d=32) == UNSUP and f(dtype=7) == UNSUP
        assert f(past=None, host=-1) == VALUE
        assert f(k=P + 8) == VALUE
    assert split(qkv=None) == NULLP and split(parts=P) == NULLP
    assert split(qkv=None, parts=P, n_parts=0) == SHAPE
    assert split(ln=float("nan")) == VALUE
    assert att(o=None) == NULLP
    for kw in (dict(new=-1), dict(keys=-1), dict(scale=0.0), dict(scale=float("inf"))):
        assert att(**kw) == VALUE, kw
    # no GPU work without tokens
    assert att(t=0) == OK and split(t=0) == OK and att(new=0) == OK

    ws = L.teeny_paged_attention_workspace_bytes
    assert ws(1, 1, 1, 4000, 8, 2, 128, BF16) > 0
    assert ws(0, 1, 1, 4000, 8, 2, 128, BF16) == 0 and ws(1, 1, 1, 4000, 8, 3, 128, BF16) == 0
    assert att(b=1, t=1, keys=4000, width=300, ld=300, ws=None) == WS
    assert att(b=1, t=1, keys=4000, width=300, ld=300, size=16) == WS
    assert att(b=1, t=1, keys=4000, width=300, ld=300, ws=P + 8) == VALUE

    def copy(src, dst, n=None, **kw):
        a = dict(pages=P, planes=2, plane=16 * 512, page=512, n_pages=16)
        a.update(kw)
        ints = ctypes.c_int32 * len(src)
        return L.teeny_copy_pages(*a.values(), ints(*src), ints(*dst), len(src) if n is None else n, None)

    assert copy([], []) == OK
    assert copy([1], [2], pages=None) == NULLP
    assert L.teeny_copy_pages(P, 2, 16 * 512, 512, 16, None, None, 1, None) == NULLP
    for kw in (dict(planes=0), dict(planes=1 << 17), dict(n_pages=0), dict(n=-1), dict(page=0), dict(plane=512)):
        assert copy([1], [2], **kw) == SHAPE, kw
    assert copy([1], [2], pages=P + 8) == VALUE and copy([1], [2], page=8) == VALUE
    for src, dst in (([16], [1]), ([-1], [1]), ([1], [16]), ([1], [-1]), ([1, 2], [3, 3]), ([1, 2], [2, 3]), ([4], [4])):
        assert copy(src, dst) == VALUE, (src, dst)


def test_paged_ops_refuse_host_tensors():
    import torch

    from teenyformers_amd import ops
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    table = torch.zeros((1, 2), dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.paged_attention(torch.zeros((1, 4, 64), dtype=torch.bfloat16), k, k, table, 0)
    with pytest.raises(ValueError):
        ops.paged_qkv_rope_split(torch.zeros((1, 512), dtype=torch.bfloat16), k, k, table, 0, 4, 1e4)
    with pytest.raises(ValueError):
        ops.copy_pages(k, [0], [1])


def test_verify_drafts_validation(L):
    def verify(**kw):
        a = dict(target=P, t_seq=400, t_row=100, draft=P, d_seq=300, d_row=100, drafts=P, u=P, b=2, k=3, cols=100,
                 t=1.0, ts=None, tokens=P, accepted=P, dtype=BF16, ws=P, size=1 << 30)
        a.update(kw)
        return L.teeny_verify_drafts(*a.values(), None)

    for name in ("target", "drafts", "u", "tokens", "accepted"):
        assert verify(**{name: None}) == NULLP, name
    assert verify(dtype=9) == UNSUP
    for kw in (dict(b=0), dict(b=-3), dict(k=0), dict(k=65), dict(cols=0), dict(cols=1 << 20), dict(t_row=99),
               dict(d_row=99), dict(t_seq=-1), dict(d_seq=-1), dict(b=1 << 15)):
        assert verify(**kw) == SHAPE, kw
    for kw in (dict(target=P + 1), dict(draft=P + 1), dict(t=-1.0), dict(t=float("nan")), dict(ws=P + 8)):
        assert verify(**kw) == VALUE, kw
    assert verify(ws=None) == WS and verify(size=64) == WS
    ws = L.teeny_verify_drafts_workspace_bytes
    assert ws(2, 3, 100, 1) > 0 and ws(2, 65, 100, 1) == 0 and ws(0, 3, 100, 0) == 0 and ws(1 << 15, 3, 100, 0) == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_paged_workspace_is_enough(L, dtype):
    """The bytes asked for with the arguments of a call are enough for it, also where max_new is
    above the tokens, or above the new tokens of each without starts."""
    import random

    import torch
    if torch.cuda.is_available():
        pytest.skip("a call that no check refuses would launch")
    rng = random.Random(dtype)
    ws = L.teeny_paged_attention_workspace_bytes

    def att(b, t, new, keys, hq, hkv, d, starts, size):
        # (a misaligned workspace: refused behind the check of its size, before any launch)
        return L.teeny_paged_attention(P, P, P, P, P, 4096, 4096, starts, P, 0, b, t, new, keys, 9, 16, hq, hkv,
                                       d, 0.1, dtype, P + 8, size, None)

    shares = 0
    for _ in range(4000):
        hkv = rng.choice([1, 2, 4, 8])
        hq, d = hkv * rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        b, each = rng.choice([1, 1, 2, 5, 16]), rng.choice([1, 1, 2, 4, 9, 40, 500])
        new, keys = rng.choice([each, each, 2 * each, 7 * each, 4096]), rng.choice([64, 500, 4000, 30000])
        a = (b, b * each, new, keys, hq, hkv, d)
        need = ws(*a, dtype)
        for starts in (None, P):
            if need == 0:
                continue  # (nothing to check it by: the call would launch)
            shares += 1
            assert att(*a, starts, need) == VALUE, a
    assert shares > 1000


def test_logit_vectors_lie_in_their_row(tmp_path):
    """Every vector that the scans of logits load lies in its row and is aligned, for rows of any
    number of columns at any offset: the loader's own arithmetic, over all its threads."""
    import os
    import shutil
    import subprocess
    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    src = os.path.join(os.path.dirname(os.path.abspath(_lib.__file__)), "csrc")
    (tmp_path / "t.cpp").write_text(r"""
#include <cstdio>
#include "chunks.h"
int main() {
  long bad = 0, n = 0;
  const int near[] = {16, 17, 23, 24, 31, 1000, 8176, 8184, 8185, 8190, 8191, 8192, 8193, 8194, 8196, 8199, 8200,
                      8208, 16377, 16383, 16384, 16385, 32000, 32768, 50257, 65536, 128255, 128256, 131072};
  for (int cols : near)
    for (int per = 4; per <= 8; per += 4)       // elements of 16 bytes: fp32, bf16
      for (int mis = 0; mis < per; ++mis)       // elements behind an aligned address
        for (int ch = 0; ch < (cols + 7 + kChunk - 1) / kChunk; ++ch)
          for (int slot = 0; slot < kChunk / kTok; ++slot, ++n) {
            const int c = ch * kChunk - mis + slot * kTok, at = vector_col(c, cols);
            if (at < 0 || at + kTok > cols || (at + mis) % per != 0) ++bad;
            if (c >= 0 && c + kTok <= cols && at != c) ++bad;
          }
  std::printf("%ld %ld\n", bad, n);
  return bad != 0;
}
""")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", src, str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert int(out.stdout.split()[1]) > 100000
