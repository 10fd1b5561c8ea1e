"""What the operators of a 4-bit transformer block refuse before any launch (no GPU needed: the
pointers are addresses that nothing may touch), and the arithmetic of their plain 64-bit forms."""
import ctypes as C
import pathlib
import re

import pytest
import torch

import mx_ref
from rfdetr_b200 import lib

INVALID = 1  # cudaErrorInvalidValue
P = 0x1000000
BIG = 2 ** 31 - 1


def test_scale_bytes():
    f = lib.lib().rfdetr_b200_mx_scale_bytes
    assert f(1, 1) == 512 and f(128, 128) == 512 and f(129, 128) == 1024 and f(128, 129) == 1024
    assert f(0, 32) == 0 and f(32, 0) == 0 and f(-1, 32) == 0
    assert f(2 ** 20, 2 ** 20) == 2 ** 35  # past 32 bits


QUANT = dict(src=P, type=1, ld=64, rows=4, k=64, codes=P, ldc=32, scales=P)


@pytest.mark.parametrize("bad", [
    dict(src=None), dict(codes=None), dict(scales=None), dict(type=2), dict(type=8), dict(type=-1), dict(rows=-1),
    dict(k=0), dict(k=-5), dict(ld=63), dict(ldc=16), dict(ldc=40), dict(codes=P + 8), dict(scales=P + 4),
    dict(src=P + 1), dict(k=65, ld=65), dict(rows=BIG), dict(k=BIG, ld=BIG, ldc=2 ** 30)])
def test_quantize_refusals(bad):
    a = {**QUANT, **bad}
    L = lib.lib()
    assert L.rfdetr_b200_op_mx_quantize(a["src"], a["type"], a["ld"], a["rows"], a["k"], a["codes"], a["ldc"],
                                        a["scales"], None) == INVALID
    assert L.rfdetr_b200_op_mx_dequantize(a["codes"], a["ldc"], a["scales"], a["rows"], a["k"], a["src"], a["type"],
                                          a["ld"], None) == INVALID


def test_nothing_to_do_succeeds():
    L = lib.lib()
    assert L.rfdetr_b200_op_mx_quantize(None, 1, 64, 0, 64, None, 0, None, None) == 0
    assert L.rfdetr_b200_op_mx_dequantize(None, 0, None, 0, 64, None, 1, 64, None) == 0
    assert L.rfdetr_b200_op_mx_gemm(None, 32, None, None, 32, None, 0, 64, 64, 0, None, None, 1, 64, None) == 0
    assert L.rfdetr_b200_op_mx_gemm(None, 32, None, None, 32, None, 64, 0, 64, 0, None, None, 1, 64, None) == 0
    assert L.rfdetr_b200_op_block_norm(lib.BlockNorm(rows=0, dim=8, type=1), None) == 0
    for seqs, tokens, longest in ((0, 8, 8), (1, 0, 8), (1, 8, 0)):
        assert L.rfdetr_b200_op_attention_packed(None, None, None, 64, 64, 64, None, 64, 1, None, seqs, tokens,
                                                 longest, 1, 1, 64, 0, 0.125, None) == 0


GEMM = dict(a=P, lda=32, sa=P, b=P, ldb=32, sb=P, M=4, N=8, K=64, act=0, bias=P, out=P, type=1, ldo=8)


@pytest.mark.parametrize("bad", [
    dict(a=None), dict(b=None), dict(sa=None), dict(sb=None), dict(out=None), dict(lda=16), dict(ldb=16),
    dict(lda=40), dict(ldb=40), dict(a=P + 8), dict(b=P + 8), dict(sa=P + 8), dict(sb=P + 8), dict(M=-1), dict(N=-1),
    dict(K=0), dict(K=-64), dict(K=65), dict(act=4), dict(act=-1), dict(type=8), dict(ldo=7), dict(out=P + 1),
    dict(bias=P + 2), dict(M=BIG), dict(N=BIG, ldo=BIG), dict(K=BIG), dict(K=2 ** 27 + 1, lda=2 ** 27, ldb=2 ** 27)])
def test_gemm_refusals(bad):
    a = {**GEMM, **bad}
    assert lib.lib().rfdetr_b200_op_mx_gemm(a["a"], a["lda"], a["sa"], a["b"], a["ldb"], a["sb"], a["M"], a["N"],
                                            a["K"], a["act"], a["bias"], a["out"], a["type"], a["ldo"],
                                            None) == INVALID


NORM = dict(y=P, resid=P, post_w=P, post_b=P, gate=P, pre_w=P, pre_b=P, out_resid=P, out=P, mx_codes=P, mx_scales=P,
            rows=4, dim=64, type=1, resid_type=0, post=1, pre=1, ldy=64, ld_resid=64, ld_out_resid=64, ld_out=64,
            ld_mx=32, ld_gate=64, gate_period=2, resid_scale=1.0, post_eps=1e-5, pre_eps=1e-5)


@pytest.mark.parametrize("bad", [
    dict(y=None), dict(post_w=None), dict(post_b=None), dict(pre_w=None), dict(pre_b=None), dict(mx_scales=None),
    dict(mx_codes=None), dict(out_resid=None, out=None, mx_codes=None, mx_scales=None), dict(rows=-1), dict(dim=0),
    dict(dim=32769, ldy=32769, ld_resid=32769, ld_out_resid=32769, ld_out=32769, ld_mx=16400, ld_gate=32769),
    dict(type=8), dict(resid_type=30), dict(resid_type=2), dict(post=3), dict(pre=-1), dict(ldy=63),
    dict(ld_resid=63), dict(ld_out_resid=63), dict(ld_out=63), dict(ld_mx=16), dict(ld_mx=36), dict(ld_gate=63),
    dict(gate_period=-1), dict(mx_codes=P + 8), dict(mx_scales=P + 8), dict(y=P + 1), dict(resid=P + 2),
    dict(gate=P + 2), dict(post_eps=-1.0), dict(pre_eps=float("nan")), dict(rows=BIG)])
def test_block_norm_refusals(bad):
    assert lib.lib().rfdetr_b200_op_block_norm(lib.BlockNorm(**{**NORM, **bad}), None) == INVALID


def test_block_norm_null_arguments():
    assert lib.lib().rfdetr_b200_op_block_norm(None, None) == INVALID


ATTN = dict(q=P, k=P, v=P, ldq=256, ldk=128, ldv=128, o=P, ldo=256, type=1, cu=P, seqs=2, tokens=16, longest=16,
            heads=4, kv=2, d=64, causal=1, scale=0.125)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(cu=None), dict(q=P + 8), dict(k=P + 2), dict(v=P + 8),
    dict(o=P + 4), dict(cu=P + 1), dict(ldq=248), dict(ldk=120), dict(ldv=120), dict(ldo=248), dict(ldq=260),
    dict(ldk=132), dict(ldv=132), dict(ldo=260), dict(type=0), dict(type=8), dict(seqs=-1), dict(tokens=-1),
    dict(longest=-1), dict(longest=2 ** 25 + 1), dict(heads=0), dict(kv=0), dict(kv=3), dict(heads=258, kv=2, ldq=258 * 64, ldo=258 * 64),
    dict(d=32), dict(d=96), dict(d=256), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(scale=2.5e38)])
def test_attention_refusals(bad):
    a = {**ATTN, **bad}
    assert lib.lib().rfdetr_b200_op_attention_packed(
        a["q"], a["k"], a["v"], a["ldq"], a["ldk"], a["ldv"], a["o"], a["ldo"], a["type"], a["cu"], a["seqs"],
        a["tokens"], a["longest"], a["heads"], a["kv"], a["d"], a["causal"], C.c_float(a["scale"]), None) == INVALID


def test_reference_rounding():
    """The plain form's own rounding at every tie, by the definition: to the even code."""
    ties = {0.25: 0, 0.75: 2, 1.25: 2, 1.75: 4, 2.5: 4, 3.5: 6, 5.0: 6, 7.9: 7, 6.0: 7}
    x = torch.zeros(len(ties), 32, dtype=torch.float64)
    for i, t in enumerate(ties):
        x[i, 0], x[i, 1], x[i, 2] = t, 4.0, -t  # the block's scale is 1
    codes, scale = mx_ref.quantize(x)
    assert codes[:, 0].tolist() == list(ties.values()) and (scale == 127).all()
    assert codes[:, 2].tolist() == [c + 8 for c in ties.values()]
    back = mx_ref.values(mx_ref.unpack(mx_ref.pack(codes)), scale)
    assert (back[:, 0] == torch.tensor(mx_ref.GRID, dtype=torch.float64)[list(ties.values())]).all()


def test_reference_scale_tiles():
    s = torch.arange(3 * 130 * 5 % 251, 3 * 130 * 5 % 251 + 130 * 5).remainder(251).to(torch.uint8).view(130, 5)
    t = mx_ref.tile_scales(s)
    assert t.numel() == lib.lib().rfdetr_b200_mx_scale_bytes(130, 5 * 32)
    assert t[(1 * 2 + 1) * 512 + 1 * 16 + 0 * 4 + 0] == s[129, 4]
    assert t[(0 * 2 + 0) * 512 + 5 * 16 + 2 * 4 + 3] == s[69, 3]


@pytest.mark.parametrize("name", ["mx.cuh", "mx_quant.cu", "mx_gemm.cu", "block_norm.cu", "attention_packed.cu"])
def test_kernels_that_start_early_read_memory_by_plain_loads(name):
    """These kernels are there while earlier ones still write what they will read, so nothing they read may be
    declared constant for their lifetime: no read-only loads, no pointers that promise it to the compiler."""
    source = (pathlib.Path(lib.__file__).parents[1] / "csrc" / name).read_text()
    code = re.sub(r"//[^\n]*", "", source)
    for word in ("__ldg", "__restrict", "ld.global.nc"):
        assert word not in code, word
    if name != "mx.cuh":
        assert "launch_early(" in code
        # every kernel waits for the work before it
        assert len(re.findall(r"\bwait_previous\(\)", code)) == len(re.findall(r"__global__", code)) > 0


def _kernel(name, kernel):
    """The text of a kernel in csrc/, comments left out."""
    source = (pathlib.Path(lib.__file__).parents[1] / "csrc" / name).read_text()
    code = re.sub(r"//[^\n]*", "", source)
    at = code.index(kernel + "(")
    return code[at:code.index("\n}\n", at)]


def test_split_product_sums_are_whole_or_not_announced():
    """The issuing warp tells the epilogue that the sums are there (a commit to `done`, once) only where no wait
    for a stage ran out: the loop over the stages keeps what each wait said, and the commit asks for it."""
    code = _kernel("mx_gemm.cu", "k_mx_gemm_few")
    assert code.count("umma_commit(done)") == 1
    guard = re.search(r"if \((\w+)\) umma_commit\(done\)", code)
    assert guard
    kept = guard.group(1)
    assert re.search(kept + r" = mbar_wait\(&full\[s\], phase, cta_abort, [^;]*;\s*if \(!" + kept + r"\) break;", code)


@pytest.mark.parametrize("name,kernel", [("mx_gemm.cu", "k_mx_gemm"), ("mx_gemm.cu", "k_mx_gemm_few"),
                                         ("attention_packed.cu", "k_attn_packed")])
def test_a_wait_that_runs_out_is_reported(name, kernel):
    """Every bounded wait sets the CTA's word, and behind the CTA's last barrier that word goes to the device's."""
    code = _kernel(name, kernel)
    waits = re.findall(r"\bmbar_wait(?:<\w+>)?\([^;]*?, cta_abort, nullptr\)", code)
    assert len(waits) == len(re.findall(r"\bmbar_wait\b", code)) >= 4
    assert len(re.findall(r"__syncthreads\(\);\s*report_abort\(cta_abort, p\.err\);", code)) == 1
    assert "__syncthreads" not in code[code.index("report_abort"):] and "return;" not in code


def test_error_word_refusal():
    assert lib.lib().rfdetr_b200_op_error_word(None) == INVALID


def test_sums_too_long_for_f32_are_refused():
    """Where the tensor core's cuts of its f32 sums would pass half a step of bf16: K above 2^21 (2^-23 for each
    64), sequences above 2^19 (2^-23 for each 16 keys)."""
    L = lib.lib()
    k = 2 ** 21 + 1
    assert L.rfdetr_b200_op_mx_gemm(P, 2 ** 21, P, P, 2 ** 21, P, 1, 1, k, 0, None, P, 0, 1, None) == INVALID
    assert L.rfdetr_b200_op_attention_packed(P, P, P, 64, 64, 64, P, 64, 1, P, 1, 2 ** 20, 2 ** 19 + 1, 1, 1, 64, 0, 0.125,
                                             None) == INVALID


@pytest.mark.parametrize("name,kernel,before", [
    ("mx_gemm.cu", "k_mx_gemm", r"tc_fence_before\(\);\s*if constexpr \(CTA2\) cluster_sync\(\);\s*else __syncthreads\(\);"),
    ("mx_gemm.cu", "k_mx_gemm_few", r"__syncwarp\(\);\s*if \(parts > 1\) \{\s*cluster_sync\(\);\s*linger_if_aborted\(cta_abort\);"),
    ("attention_packed.cu", "k_attn_packed", r"tc_fence_before\(\);\s*__syncthreads\(\);")])
def test_a_cta_that_gives_up_waits_for_what_is_in_flight(name, kernel, before):
    """Behind the roles, in front of the barrier that ends in freeing tensor memory and leaving (and behind the
    cluster's, where others send to this CTA)."""
    code = _kernel(name, kernel)
    at = re.search(r"linger_if_aborted\(cta_abort\);\s*" + before, code)
    assert at and code.rindex("mbar_wait") < at.start() < code.index("report_abort") < code.index("tmem_dealloc")
