"""The serving entries without a GPU: exported symbols, struct layouts, and
the refusals, which come before any CUDA call."""
import ctypes as C
import os
import re
import subprocess

import pytest

from akili_bench_b200 import abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 0x10000  # any aligned address: refused calls touch nothing


def test_header_symbols_and_layouts(tmp_path):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "akili_serving.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(akili_\w+)\s*\(", text))
    assert names == {f"akili_{n}" for n in abi.SERVING_OPS} | {"akili_tree_attention_workspace"}
    L = abi.load()
    for n in names:
        assert getattr(L, n) is not None
    src = '#include "akili_serving.h"\n#include <stdio.h>\nint main(void) {\n'
    structs = sorted({(n.replace("rope_append", "rope"), st) for n, (st, _) in abi.SERVING_OPS.items()}, key=lambda x: x[0])
    for n, st in structs:
        src += f'printf("{n} %zu\\n", sizeof(akili_{n}_arg_t));\n'
    (tmp_path / "s.c").write_text(src + "return 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "s.c", "-o", "s"],
                   cwd=tmp_path, check=True)
    out = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout
    sizes = dict(ln.split() for ln in out.splitlines())
    for n, (st, size) in abi.SERVING_OPS.items():
        assert int(sizes[n.replace("rope_append", "rope")]) == size == C.sizeof(st), n


def code(op, arg):
    return getattr(abi.load(), f"akili_{op}")(C.byref(arg) if arg is not None else None, None)


def rope_arg(**kw):
    a = abi.RopeArg(abi.DTYPE_F16, 0, 4, 8, 2, 64, 64, 100, A, A, A, A, A, A, 512, 64, 128, 64, 512, 64, 128, 64, A, A, A,
                    A, 10, 16, 128, 64, 2048, 128, 64, 2048, 128, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("op,change,want", [
    ("rope", {"dtype": 3}, abi.E_DTYPE), ("rope", {"flags": 4}, abi.E_UNSUPPORTED),
    ("rope", {"rot_dim": 0}, abi.E_SHAPE), ("rope", {"rot_dim": 63}, abi.E_SHAPE), ("rope", {"rot_dim": 66}, abi.E_SHAPE),
    ("rope", {"max_positions": 0}, abi.E_SHAPE), ("rope", {"tokens": 1 << 31}, abi.E_SHAPE),
    ("rope", {"q_addr": 0}, abi.E_NULL_ARG), ("rope", {"k_out_addr": 0}, abi.E_NULL_ARG),
    ("rope", {"positions_addr": 0}, abi.E_NULL_ARG), ("rope", {"table_addr": A + 2}, abi.E_ALIGN),
    ("rope", {"k_addr": A + 1}, abi.E_ALIGN), ("rope", {"tokens": 0, "q_addr": 0}, abi.OK),
    ("rope_append", {"slots_addr": 0}, abi.E_NULL_ARG), ("rope_append", {"slots_addr": A + 4}, abi.E_ALIGN),
    ("rope_append", {"v_addr": 0}, abi.E_NULL_ARG), ("rope_append", {"page_size": 0}, abi.E_SHAPE)])
def test_rope_refusals(op, change, want):
    assert code(op, rope_arg(**change)) == want


def test_null_blocks_are_refused():
    for op in abi.SERVING_OPS:
        assert code(op, None) == abi.E_NULL_ARG


def table_arg(**kw):
    a = abi.RopeTableArg(100, 64, 0, 0, 10000.0, 2.0, 4096.0, 1.0, 4.0, 0.0, A)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,want", [
    ({"scaling": 5}, abi.E_UNSUPPORTED), ({"rot_dim": 258}, abi.E_SHAPE), ({"rot_dim": 3}, abi.E_SHAPE),
    ({"max_positions": 0}, abi.E_SHAPE), ({"base": 0.0}, abi.E_UNSUPPORTED), ({"base": float("nan")}, abi.E_UNSUPPORTED),
    ({"scaling": 1, "factor": 0.0}, abi.E_UNSUPPORTED), ({"scaling": 2, "rot_dim": 2}, abi.E_UNSUPPORTED),
    ({"scaling": 3, "original_positions": 0.0}, abi.E_UNSUPPORTED), ({"scaling": 4, "high": 1.0}, abi.E_UNSUPPORTED),
    ({"scaling": 4, "base": 1.0}, abi.E_UNSUPPORTED), ({"amplitude": -1.0}, abi.E_UNSUPPORTED),
    ({"reserved": 1}, abi.E_UNSUPPORTED), ({"table_addr": 0}, abi.E_NULL_ARG), ({"table_addr": A + 2}, abi.E_ALIGN)])
def test_rope_table_refusals(change, want):
    assert code("rope_table", table_arg(**change)) == want


def prompt_arg(**kw):
    a = abi.PromptAttentionArg(abi.DTYPE_F16, 8, 2, 64, 3, 100, 100, 1, 0.0, 0, A, A, A, A, 0, A, A, 512, 64, 128, 64,
                               128, 64, 512, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def tree_arg(**kw):
    a = abi.TreeAttentionArg(abi.DTYPE_BF16, 8, 2, 64, 3, 10, 50, 16, 7, 0, 0.0, 0, A, A, A, A, 0, A, A, A, 0, 0, 0, 512,
                             64, 512, 64, 2048, 128, 64, 2048, 128, 64, 7, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


ATTENTION = [
    ({"dtype": abi.DTYPE_F32}, abi.E_DTYPE), ({"q_heads": 0}, abi.E_SHAPE), ({"kv_heads": 3}, abi.E_SHAPE),
    ({"head_dim": 0}, abi.E_SHAPE), ({"head_dim": 60}, abi.E_SHAPE), ({"head_dim": 136}, abi.E_UNSUPPORTED),
    ({"softmax_scale": -1.0}, abi.E_UNSUPPORTED), ({"softmax_scale": float("nan")}, abi.E_UNSUPPORTED),
    ({"softmax_scale": float("inf")}, abi.E_UNSUPPORTED), ({"reserved": 1}, abi.E_UNSUPPORTED),
    ({"batch": 0}, abi.E_SHAPE), ({"total_q": (1 << 30) + 1}, abi.E_SHAPE), ({"total_q": 0, "q_addr": 0}, abi.OK),
    ({"q_addr": 0}, abi.E_NULL_ARG), ({"o_addr": 0}, abi.E_NULL_ARG), ({"q_addr": A + 8}, abi.E_ALIGN),
    ({"lse_addr": A + 2}, abi.E_ALIGN), ({"cu_q_addr": 0}, abi.E_NULL_ARG), ({"q_stride_token": 516}, abi.E_ALIGN),
    ({"o_stride_head": 4}, abi.E_ALIGN), ({"q_stride_head": 0}, abi.E_SHAPE), ({"q_stride_token": -512}, abi.E_SHAPE)]


@pytest.mark.parametrize("change,want", ATTENTION + [
    ({"causal": 2}, abi.E_UNSUPPORTED), ({"k_addr": 0}, abi.E_NULL_ARG), ({"cu_k_addr": 0}, abi.E_NULL_ARG),
    ({"cu_k_addr": A + 2}, abi.E_ALIGN), ({"k_stride_head": 60}, abi.E_ALIGN), ({"v_stride_token": 12}, abi.E_ALIGN),
    ({"k_stride_head": 0}, abi.E_SHAPE)])
def test_prompt_attention_refusals(change, want):
    assert code("prompt_attention", prompt_arg(**change)) == want


@pytest.mark.parametrize("change,want", ATTENTION + [
    ({"page_size": 12}, abi.E_SHAPE), ({"page_size": 0}, abi.E_SHAPE), ({"max_pages": 0}, abi.E_SHAPE),
    ({"num_pages": 0}, abi.E_SHAPE), ({"max_pages": 1 << 28}, abi.E_SHAPE), ({"k_pages_addr": 0}, abi.E_NULL_ARG),
    ({"v_pages_addr": A + 2}, abi.E_ALIGN), ({"page_table_addr": 0}, abi.E_NULL_ARG),
    ({"context_lens_addr": A + 1}, abi.E_ALIGN), ({"mask_addr": A}, abi.E_SHAPE),
    ({"mask_addr": A + 1, "mask_words": 1}, abi.E_ALIGN), ({"k_page_stride_token": 100}, abi.E_ALIGN),
    ({"v_page_stride_page": 4}, abi.E_ALIGN), ({"v_page_stride_head": 0}, abi.E_SHAPE),
    ({"k_page_stride_page": -2048}, abi.E_SHAPE)])
def test_tree_attention_refusals(change, want):
    assert code("tree_attention", tree_arg(**change)) == want


@pytest.mark.parametrize("change,want", [
    ({"reserved": 1}, abi.E_UNSUPPORTED), ({"mask_words": 0}, abi.E_SHAPE), ({"batch": 0}, abi.E_SHAPE),
    ({"parents_addr": 0}, abi.E_NULL_ARG), ({"mask_addr": A + 2}, abi.E_ALIGN), ({"total_q": 0}, abi.OK)])
def test_tree_mask_refusals(change, want):
    a = abi.TreeMaskArg(2, 10, 1, 0, A, A, A)
    for k, v in change.items():
        setattr(a, k, v)
    assert code("tree_mask", a) == want


@pytest.mark.parametrize("change,want", [
    ({"elem_bytes": 8}, abi.E_DTYPE), ({"reserved": 1}, abi.E_UNSUPPORTED), ({"layers": 0}, abi.E_SHAPE),
    ({"batch": 65536}, abi.E_SHAPE), ({"page_size": 0}, abi.E_SHAPE), ({"kv_heads": 0}, abi.E_SHAPE),
    ({"k_pages_addr": 0}, abi.E_NULL_ARG), ({"v_pages_addr": A + 1}, abi.E_ALIGN), ({"accepted_addr": 0}, abi.E_NULL_ARG),
    ({"n_accepted_addr": A + 2}, abi.E_ALIGN), ({"new_lens_addr": 2 * A + 1}, abi.E_ALIGN),
    ({"new_lens_addr": A}, abi.E_UNSUPPORTED), ({"batch": 0, "k_pages_addr": 0}, abi.OK)])
def test_cache_accept_refusals(change, want):
    a = abi.CacheAcceptArg(2, 4, 3, 2, 64, 50, 16, 7, 8, 0, A, A, A, A, A, A, 2 * A, 102400, 2048, 128, 64, 102400, 2048,
                           128, 64, 7, 8)
    for k, v in change.items():
        setattr(a, k, v)
    assert code("cache_accept", a) == want


@pytest.mark.parametrize("read,cols,stride", [("context_lens", 1, 0), ("n_accepted", 1, 0), ("accepted", 8, 11),
                                              ("page_table", 7, 11)])
def test_cache_accept_refuses_new_lengths_over_what_it_reads(read, cols, stride):
    """New lengths (batch int32) that share even four bytes with an index tensor; next to it they are taken."""
    torch = pytest.importorskip("torch")
    batch = 3
    first, last = (0, 4 * (batch - 1)) if stride == 0 else (0, 4 * ((batch - 1) * stride + cols - 1))
    for at, refused in ((first, True), (last, True), (first - 4 * (batch - 1), True), (first - 4 * batch, False),
                        (last + 4, False), (4 * cols, stride == 0)):
        a = abi.CacheAcceptArg(2, 4, batch, 2, 64, 50, 16, 7, 8, 0, A, A, 2 * A, 3 * A, 4 * A, 5 * A, 0, 102400, 2048, 128,
                               64, 102400, 2048, 128, 64, 11, 11)
        a.new_lens_addr = getattr(a, read + "_addr") + at
        if refused:
            assert code("cache_accept", a) == abi.E_UNSUPPORTED, (read, at)
        elif not torch.cuda.is_available():  # (with a GPU it would run, on addresses that are none)
            assert code("cache_accept", a) == abi.E_NO_DEVICE, (read, at)


def accept_arg(**kw):
    a = abi.CacheAcceptArg(2, 4, 3, 2, 64, 50, 16, 7, 8, 0, A, A, A, A, A, A, 2 * A, 102400, 2048, 128, 64, 102400, 2048,
                           128, 64, 7, 8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("op,make,extents", [
    ("rope", rope_arg, {"q_out_stride_token": "tokens", "q_out_stride_head": "q_heads", "k_out_stride_token": "tokens",
                        "k_out_stride_head": "k_heads"}),
    ("rope_append", rope_arg, {"q_out_stride_head": "q_heads", "k_out_stride_token": "tokens",
                               "k_page_stride_page": "num_pages", "k_page_stride_token": "page_size",
                               "v_page_stride_token": "page_size", "v_page_stride_head": "k_heads"}),
    ("prompt_attention", prompt_arg, {"o_stride_token": "total_q", "o_stride_head": "q_heads"}),
    ("tree_attention", tree_arg, {"o_stride_token": "total_q", "o_stride_head": "q_heads"}),
    ("cache_accept", accept_arg, {"k_page_stride_layer": "layers", "k_page_stride_page": "num_pages",
                                  "v_page_stride_token": "page_size", "v_page_stride_head": "kv_heads"})])
def test_outputs_whose_entries_lie_over_one_another_are_refused(op, make, extents):
    """Stride 0 along a written axis; along an axis of one entry it is never used."""
    torch = pytest.importorskip("torch")
    for stride, extent in extents.items():
        assert code(op, make(**{stride: 0})) == abi.E_SHAPE, stride
        if not torch.cuda.is_available():
            one = {extent: 1}
            if extent == "q_heads" and op.endswith("attention"):
                one["kv_heads"] = 1
            if extent == "page_size" and op == "cache_accept":
                one["max_pages"] = 1
            assert code(op, make(**{stride: 0}, **one)) == abi.E_NO_DEVICE, stride


def test_valid_blocks_without_a_gpu_report_no_device():
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert code("rope", rope_arg()) == abi.E_NO_DEVICE
    assert code("prompt_attention", prompt_arg()) == abi.E_NO_DEVICE
    assert code("tree_attention", tree_arg()) == abi.E_NO_DEVICE


def test_front_end_refuses_cpu_tensors_and_wrong_types():
    torch = pytest.importorskip("torch")
    from akili_bench_b200 import ops
    q = torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        ops.prompt_attention(q, q, q, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.rope_table(10, 64, scaling="cubic")


def test_the_front_end_is_rebuilt_when_what_it_is_made_of_changes(tmp_path):
    """Its source, every header that it includes from here, and torch itself."""
    torch = pytest.importorskip("torch")
    from akili_bench_b200 import build
    names = {os.path.realpath(p) for p in build._serving_sources()}
    seen, todo = set(), [os.path.join(build.CSRC, "serving_torch.cpp")]
    while todo:
        path = os.path.realpath(todo.pop())
        if path in seen:
            continue
        seen.add(path)
        for h in re.findall(r'^#include "([^"]+)"', open(path).read(), flags=re.M):
            todo.append(os.path.join(os.path.dirname(path), h))
    assert seen <= names
    assert os.path.realpath(os.path.join(os.path.dirname(torch.__file__), "version.py")) in names
    out = tmp_path / "module.so"
    out.touch()
    for name in names:
        os.utime(out, (os.path.getmtime(name) - 1,) * 2)
        assert build._stale(str(out), [name])
