"""The serving operators where calls meet: waits that give up, streams, captured
graphs, buffers that overlap, requests a default could hide."""
import ctypes as C
import os
import subprocess
import sys
import threading

import pytest

torch = pytest.importorskip("torch")

from akili_bench_b200 import abi, ops  # noqa: E402
import serving_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731


@pytest.fixture(autouse=True)
def clean_status():
    ops.device_status()
    yield
    assert ops.device_status() == 0


@pytest.mark.parametrize("limit_us", [200, 5000])
def test_warps_that_share_a_barrier_give_up_together(limit_us):
    """One warp's limit passes before the phase completes, the other's does not: neither goes on (it would wait
    for the other at their next barrier); the status would be STATUS_SELFTEST_SHARED."""
    ops.selftest_wait_timeout(limit_us)
    assert ops.device_status() == ops.STATUS_SELFTEST


def test_a_timeout_is_reported_after_a_skipped_index():
    """A skipped index is survivable, a wait that gave up is not: whichever comes first, the latter is reported."""
    q = torch.ones(2, 1, 8, device="cuda", dtype=F16)
    table = ops.rope_table(4, 8)
    skip = lambda: ops.rope(q, q, i32([0, 9]), table)  # noqa: E731
    wait = lambda: ops.selftest_wait_timeout(200)  # noqa: E731
    v = C.c_uint32(0)
    for calls, status, rc in (((skip,), abi.STATUS_BAD_INDEX, abi.E_SHAPE),
                              ((skip, wait), ops.STATUS_SELFTEST, abi.E_DEVICE_TIMEOUT),
                              ((wait, skip), ops.STATUS_SELFTEST, abi.E_DEVICE_TIMEOUT),
                              ((skip, wait, skip), ops.STATUS_SELFTEST, abi.E_DEVICE_TIMEOUT)):
        for call in calls:
            call()
        assert abi.load().akili_device_status(C.byref(v), 1) == rc and v.value == status
    assert ops.device_status() == 0


# ------------------------------------------------------- streams and graphs --
TOKENS, HEADS, DIM = 1024, 32, 128


def side_calls():
    """name -> (call on a stream, bytes of its result), on inputs that are ready."""
    q = torch.randn(TOKENS, HEADS, DIM, device="cuda", dtype=F16)
    none = q[:, :0]
    positions = torch.arange(TOKENS, dtype=torch.int32, device="cuda")
    table = ops.rope_table(TOKENS, DIM)
    pages, v_pages = (torch.zeros(TOKENS // 16, 16, 1, DIM, device="cuda", dtype=F16) for _ in range(2))
    out = torch.empty_like(q)
    slots = torch.arange(TOKENS, device="cuda")
    cu, lens = i32([0, TOKENS]), i32([0])
    page_table = torch.arange(TOKENS // 16, dtype=torch.int32, device="cuda")[None]
    parents = torch.arange(TOKENS, dtype=torch.int32, device="cuda") - 1
    many = torch.zeros(1 << 15, dtype=torch.int32, device="cuda")
    one_page, v_page = (torch.zeros(1, 8, 1, 8, device="cuda", dtype=F16) for _ in range(2))
    wide = torch.zeros(1 << 15, 1, dtype=torch.int32, device="cuda")
    of = lambda t: t[0] if isinstance(t, tuple) else t  # noqa: E731
    return {
        "rope": (lambda s: of(ops.rope(q, none, positions, table, stream=s)), q.nbytes),
        "rope_append": (lambda s: ops.rope_append(q, q[:, :1], q[:, :1], positions, table, slots, pages, v_pages,
                                                  stream=s), q.nbytes),
        "rope_table": (lambda s: ops.rope_table(TOKENS, DIM, stream=s), TOKENS * DIM * 4),
        "prompt_attention": (lambda s: ops.prompt_attention(q, q, q, cu, stream=s), q.nbytes),
        "prompt_lse": (lambda s: ops.prompt_attention(q, q, q, cu, out=out, return_lse=True, stream=s)[1],
                       TOKENS * HEADS * 4),
        "tree_attention": (lambda s: ops.tree_attention(q, pages, pages, page_table, lens, cu, stream=s), q.nbytes),
        "tree_mask": (lambda s: ops.tree_mask(parents, cu, TOKENS, stream=s), TOKENS * TOKENS // 8),
        "cache_accept": (lambda s: ops.cache_accept(one_page, v_page, wide, many, wide, many, stream=s),
                         many.nbytes),
    }


@pytest.mark.parametrize("name", ["rope", "rope_append", "rope_table", "prompt_attention", "prompt_lse",
                                  "tree_attention", "tree_mask", "cache_accept"])
def test_results_on_another_stream_do_not_take_memory_that_is_still_in_use(name):
    """A block freed on the current stream, while what is queued there has yet to read it, is not the result of a
    call on a stream that waits for nothing."""
    call, size = side_calls()[name]
    side = torch.cuda.Stream()
    call(side)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    blocks = [torch.full((size,), 7, dtype=torch.uint8, device="cuda") for _ in range(4)]
    kept = [torch.zeros_like(b) for b in blocks]
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)  # some 50 ms
    for b, k in zip(blocks, kept):
        k.copy_(b)
    freed = {b.data_ptr() for b in blocks}
    del blocks, b, k
    result = call(side)
    assert result.data_ptr() not in freed
    torch.cuda.synchronize()
    assert all((k == 7).all() for k in kept)


def test_results_on_another_stream_outlive_what_the_callers_stream_does_with_them():
    """Freed while the caller's stream has yet to read it, a result's memory does not go to that stream's next call."""
    call, size = side_calls()["rope"]
    side = torch.cuda.Stream()
    result = call(side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(100_000_000)
    kept = result.clone()
    freed = result.data_ptr()
    del result
    later = call(side)
    assert later.data_ptr() != freed
    torch.cuda.synchronize()
    assert torch.equal(kept, later)


def test_streams_of_other_kinds():
    q = torch.randn(4, 2, 64, device="cuda", dtype=F16)
    cu = i32([0, 4])
    want = ops.prompt_attention(q, q, q, cu)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    raw = type("Raw", (), {"cuda_stream": side.cuda_stream})()
    for s in (side, raw, torch.cuda.ExternalStream(side.cuda_stream), torch.cuda.default_stream()):
        got = ops.prompt_attention(q, q, q, cu, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    with torch.cuda.stream(side):
        got = ops.prompt_attention(q, q, q, cu, stream=torch.cuda.default_stream())
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    with pytest.raises(ValueError):
        ops.prompt_attention(q, q, q, cu, stream=torch.Stream("cpu"))
    with pytest.raises(AttributeError):
        ops.prompt_attention(q, q, q, cu, stream=3)


def step(tokens, group, context, dtype=F16, pages=64):
    """Arguments of a tree_attention call of `tokens` new tokens for each of two sequences."""
    q = torch.randn(2 * tokens, group, 128, device="cuda", dtype=dtype)
    kp, vp = (torch.randn(2 * pages, 16, 1, 128, device="cuda", dtype=dtype) for _ in range(2))
    table = torch.randperm(2 * pages, device="cuda").to(torch.int32).view(2, pages)
    return q, kp, vp, table, i32([context, context // 3]), i32([0, tokens, 2 * tokens])


def c_entry(args, out, stream, workspace=None):
    """akili_tree_attention itself, without the torch front end."""
    q, kp, vp, table, lens, cu = args
    a = abi.TreeAttentionArg(abi.DTYPE_F16, q.shape[1], 1, 128, 2, q.shape[0], kp.shape[0], 16, table.shape[1], 0, 0.0,
                             0, q.data_ptr(), kp.data_ptr(), vp.data_ptr(), out.data_ptr(), 0, table.data_ptr(),
                             lens.data_ptr(), cu.data_ptr(), 0, 0, 0, *q.stride()[:2], *out.stride()[:2],
                             *kp.stride()[:3], *vp.stride()[:3], table.stride(0), 0)
    if workspace is not None:
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.nbytes
    assert abi.load().akili_tree_attention(C.byref(a), stream.cuda_stream) == abi.OK


@pytest.mark.parametrize("front_end", [True, False])
def test_a_captured_step_outlives_the_growth_of_the_streams_scratch(front_end):
    """Captured in the 16-row form without a workspace; the 256-row form then needs a larger scratch on the same
    stream, and the memory that this frees is taken by others."""
    small, large = step(1, 8, 900), step(60, 8, 700)
    want, want_large = (ops.tree_attention(*s, workspace=torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
                        for s in (small, large))
    out = torch.zeros_like(want)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    call = (lambda: ops.tree_attention(*small, out=out)) if front_end else (lambda: c_entry(small, out, side))
    with torch.cuda.stream(side):
        call()  # the scratch of this stream, sized for the small step
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            call()
        out.zero_()
        assert torch.equal(ops.tree_attention(*large), want_large)
        junk = [torch.full((n << 20,), 255, dtype=torch.uint8, device="cuda") for n in (1, 2, 3, 4, 5, 8)]
        graph.replay()
        side.synchronize()
    assert torch.equal(out, want)
    assert all((j == 255).all() for j in junk)


def test_a_captured_step_shares_no_memory_with_the_streams_eager_calls():
    """Replays on one stream beside eager calls on the stream of the capture."""
    captured, eager = step(1, 8, 1000), step(3, 2, 800)
    want, want_eager = ops.tree_attention(*captured), ops.tree_attention(*eager)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    out = torch.zeros_like(want)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):  # (no eager call before it)
        ops.tree_attention(*captured, out=out)
    torch.cuda.synchronize()
    for _ in range(50):
        with torch.cuda.stream(other):
            graph.replay()
        with torch.cuda.stream(side):
            got = [ops.tree_attention(*eager) for _ in range(3)]
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(x, want_eager) for x in got)


# ------------------------------------------------------------------- accept --
def test_cache_accept_refuses_to_write_lengths_over_its_inputs():
    pages = torch.zeros(2, 4, 8, 1, 8, device="cuda", dtype=F16)
    ints = torch.zeros(4, 16, dtype=torch.int32, device="cuda")
    table, lens, accepted, n = ints[:2, :2], ints[2, :2], ints[:2, 4:6], ints[3, :2]
    for out in (lens, n, ints[2, 1:3], ints[3, 1:3], ints[0, 4:6], ints[1, 1:3], ints[1, 5:7]):
        with pytest.raises(abi.AkiliError) as e:
            ops.cache_accept(pages, pages.clone(), table, lens, accepted, n, new_lens=out)
        assert e.value.code == abi.E_UNSUPPORTED
    for out in (ints[3, 2:4], ints[0, 2:4], ints[0, 6:8]):  # (between the rows of the page table and of accepted)
        assert ops.cache_accept(pages, pages.clone(), table, lens, accepted, n, new_lens=out).tolist() == [0, 0]


# --------------------------------------------------- what a default could hide --
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-50])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 55])  # (scores up to 2^120, near the end of fp32)
@pytest.mark.parametrize("qlens,heads", [([40, 130], 2), ([700, 300], 32)])  # one tile a CTA, two
def test_prompt_attention_with_a_scale_of_zero(scale, size, qlens, heads):
    g = torch.Generator().manual_seed(len(qlens) * heads)
    q, k, v = (torch.randn(sum(qlens), heads, 64, generator=g) for _ in range(3))
    q, k, v = (q * size).to(BF16), (k * size).to(BF16), v.to(BF16)
    cu = [0, qlens[0], sum(qlens)]
    got, lse = ops.prompt_attention(q.cuda(), k.cuda(), v.cuda(), i32(cu), softmax_scale=scale, return_lse=True)
    for a, b in zip(cu, cu[1:]):
        o, l, bound, l_bound = ref.attend(q[a:b], k[a:b], v[a:b], ref.causal(b - a, b - a), 0.0)
        ref.assert_within(got[a:b], o, bound)
        ref.assert_within(lse[a:b], l, l_bound)


@pytest.mark.parametrize("new,group", [(1, 4), (5, 8), (20, 6), (70, 4)])  # 16, 64, 128 and 256 rows
def test_tree_attention_with_a_scale_of_zero(new, group):
    args = step(new, group, 900)
    q, kp, vp, table, lens, cu = args
    got = ops.tree_attention(*args, softmax_scale=0.0)
    for b, c in enumerate(lens.tolist()):
        k, v = (p[table[b].long()].flatten(0, 1)[:c + new].cpu() for p in (kp, vp))
        o, _, bound, _ = ref.attend(q[b * new:(b + 1) * new].cpu(), k, v, ref.causal(new, c + new), 0.0)
        ref.assert_within(got[b * new:(b + 1) * new], o, bound)


def test_a_mask_of_no_words_is_refused():
    """It says that no new token sees any; without a mask they would see one another."""
    args = step(3, 4, 100)
    with pytest.raises(ValueError):
        ops.tree_attention(*args, torch.zeros(6, 0, dtype=torch.int32, device="cuda"))
    none = (args[0][:0], *args[1:5], i32([0, 0, 0]))
    assert ops.tree_attention(*none, torch.zeros(0, 0, dtype=torch.int32, device="cuda")).shape == (0, 4, 128)


def test_scales_that_are_refused():
    q = torch.ones(4, 2, 64, device="cuda", dtype=F16)
    for scale in (-1.0, float("nan"), float("inf"), 1e39):
        with pytest.raises(abi.AkiliError) as e:
            ops.prompt_attention(q, q, q, i32([0, 4]), softmax_scale=scale)
        assert e.value.code == abi.E_UNSUPPORTED


# ----------------------------------------------------------------- gradients --
def tracked(*shape, dtype=F16):
    """A tensor that is part of a graph, and the leaf it comes from."""
    leaf = torch.randn(shape, device="cuda", dtype=dtype, requires_grad=True)
    return leaf * 1, leaf


def test_results_of_tracked_inputs_raise_in_a_backward_pass():
    q, leaf = tracked(8, 2, 64)
    plain = q.detach()
    pos, table = torch.arange(8, dtype=torch.int32, device="cuda"), ops.rope_table(8, 64)
    pages = torch.zeros(2, 16, 2, 64, device="cuda", dtype=F16)
    v_pages, slots = pages.clone(), torch.arange(8, device="cuda")
    tree = lambda x: ops.tree_attention(x, pages, v_pages, i32([[0, 1]]), i32([3]), i32([0, 8]),  # noqa: E731
                                        return_lse=True)
    calls = {
        "inverse=True": lambda x: ops.rope(x, x, pos, table),
        "rope_append": lambda x: (ops.rope_append(x, x, x, pos, table, slots, pages, v_pages),),
        "prompt_attention": lambda x: ops.prompt_attention(x, x, x, i32([0, 8]), return_lse=True),
        "tree_attention": tree,
    }
    for name, call in calls.items():
        want = call(plain)
        got = call(q)
        for y, w in zip(got, want):
            assert y.requires_grad and not w.requires_grad and torch.equal(y, w)
            with pytest.raises(RuntimeError, match=name):
                y.sum().backward(retain_graph=True)
        with torch.no_grad():
            assert not any(y.requires_grad for y in call(q))
    assert leaf.grad is None and not pages.requires_grad and not v_pages.requires_grad
    # the output of a call may be part of the graph as well
    out = torch.empty_like(plain)
    assert ops.prompt_attention(plain, q, plain, i32([0, 8]), out=out) is out and out.requires_grad
    with pytest.raises(RuntimeError, match="prompt_attention"):
        out.sum().backward()


def test_values_that_were_saved_for_a_backward_pass_are_not_overwritten_unnoticed():
    pos, table = torch.arange(8, dtype=torch.int32, device="cuda"), ops.rope_table(8, 64)
    x, _ = tracked(8, 2, 64)
    y = (x * x).sum()
    ops.rope(x, x[:, :0], pos, table, q_out=x)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    leaf = torch.randn(8, 2, 64, device="cuda", dtype=F16, requires_grad=True)
    before = leaf.detach().clone()
    with pytest.raises(RuntimeError, match="leaf"):
        ops.rope(leaf, leaf[:, :0], pos, table, q_out=leaf)
    assert torch.equal(leaf, before)
    with torch.no_grad():
        ops.rope(leaf, leaf[:, :0], pos, table, q_out=leaf)


def test_tensors_written_in_place_get_a_new_version():
    new = lambda *s: torch.zeros(s, device="cuda", dtype=F16)  # noqa: E731
    q, k, v, pages, v_pages, out = new(8, 2, 64), new(8, 2, 64), new(8, 2, 64), new(2, 16, 2, 64), new(2, 16, 2, 64), \
        new(8, 2, 64)
    pos, table, slots = torch.arange(8, dtype=torch.int32, device="cuda"), ops.rope_table(8, 64), \
        torch.arange(8, device="cuda")
    lens = i32([0])
    calls = [
        (lambda: ops.rope(q, k, pos, table, q_out=q, k_out=k), (q, k)),
        (lambda: ops.rope_append(q, k, v, pos, table, slots, pages, v_pages, q_out=out, k_out=k),
         (out, k, pages, v_pages)),
        (lambda: ops.prompt_attention(q, k, v, i32([0, 8]), out=out), (out,)),
        (lambda: ops.tree_attention(q, pages, v_pages, i32([[0, 1]]), i32([3]), i32([0, 8]), out=out), (out,)),
        (lambda: ops.cache_accept(pages, v_pages, i32([[0, 1]]), i32([3]), i32([[1]]), i32([1]), new_lens=lens),
         (pages, v_pages, lens)),
    ]
    every = (q, k, v, pages, v_pages, out, lens)
    for call, changed in calls:
        before = [t._version for t in every]
        call()
        for t, old in zip(every, before):
            assert (t._version > old) == any(t is c for c in changed)
    with torch.inference_mode():
        x = torch.zeros(8, 2, 64, device="cuda", dtype=F16)
        ops.rope(x, x[:, :0], pos, table, q_out=x)
        ops.rope(q, k, pos, table, q_out=q, k_out=k)
    ops.rope(x, x[:, :0], pos, table, q_out=x)  # (an inference tensor has no version)


# ------------------------------------------------------------ batches, order --
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,context", [([1] * 9 + [200] + [1] * 6, 300),   # 64 rows: the chunk in many items
                                         ([1, 500, 1, 1], 130),              # 256 rows: single tokens too
                                         ([1, 1, 60, 1, 1, 1, 1, 1], 700)])  # 64 rows, cut items
def test_a_chunk_among_single_tokens(dtype, new, context):
    g = torch.Generator().manual_seed(sum(new))
    heads, hk, d, page = 8, 2, 128, 16
    lens = [(context * (b + 3) * 7) % (2 * context) for b in range(len(new))]
    per = -(-max(c + n for c, n in zip(lens, new)) // page)
    table = torch.randperm(len(new) * per, generator=g).to(torch.int32).view(len(new), per)
    kp, vp = (torch.randn(len(new) * per, page, hk, d, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(sum(new), heads, d, generator=g).to(dtype)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    got, lse = ops.tree_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), i32(lens), i32(cu), return_lse=True)
    for b, (c, n) in enumerate(zip(lens, new)):
        k, v = (p[table[b].long()].flatten(0, 1)[:c + n] for p in (kp, vp))
        o, l, bound, l_bound = ref.attend(q[cu[b]:cu[b + 1]], k, v, ref.causal(n, c + n))
        ref.assert_within(got[cu[b]:cu[b + 1]], o, bound, f"sequence {b}")
        ref.assert_within(lse[cu[b]:cu[b + 1]], l, l_bound, f"lse of sequence {b}")


def test_two_threads_on_one_stream():
    """The scratch of the stream is shared, the calls of the front end take turns."""
    sizes = [step(1, 8, 900), step(60, 8, 700), step(9, 4, 400)]
    want = [ops.tree_attention(*s) for s in sizes]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    wrong = []

    def work(first):
        with torch.cuda.stream(stream):
            got = [(i % 3, ops.tree_attention(*sizes[i % 3])) for i in range(first, first + 60)]
            stream.synchronize()
            wrong.extend(i for i, o in got if not torch.equal(o, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


CHAIN = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from akili_bench_b200 import ops
g = torch.Generator("cuda").manual_seed(5)
r = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float16)
i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
pages, v_pages, table = r(40, 16, 2, 64), r(40, 16, 2, 64), ops.rope_table(512, 64)
page_table = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20)
lens, cu, out = i([0, 0]), i([0, 30, 70]), []
pos = torch.cat([torch.arange(30), torch.arange(40)]).int().cuda()
slots = torch.cat([torch.arange(30), torch.arange(40) + 320]).cuda()
q, k, v = r(70, 8, 64), r(70, 2, 64), r(70, 2, 64)
q = ops.rope_append(q, k, v, pos, table, slots, pages, v_pages, k_out=k)
out.append(ops.prompt_attention(q, k, v, cu))
lens = i([30, 40])
for s in range(20):  # each call's inputs are the results of the one before
    cu = i([0, 4, 8])
    mask = ops.tree_mask(i([-1, 0, 0, 2] * 2), cu, 4)
    base = torch.stack([lens, lens + 320], 1)
    at = (base[:, 1:] + torch.arange(4, device="cuda") + torch.tensor([[0], [0]], device="cuda"))
    at[0] -= 320
    x = out[-1][:8]
    q = ops.rope_append(x, x[:, :2], x[:, 2:4], i([0, 1, 1, 2] * 2), table, at.flatten().long(), pages, v_pages)
    out.append(ops.tree_attention(q, pages, v_pages, page_table, lens, cu, mask))
    lens = ops.cache_accept(pages, v_pages, page_table, lens, i([[0, 2, 3]] * 2), i([3, 2]))
out += [lens, pages, v_pages]
torch.save([t.cpu() for t in out], sys.argv[2])
assert ops.device_status() == 0
"""


def test_dependent_launches_give_what_plain_ones_do(tmp_path):
    """A chain of calls, each on the results of the one before, with AKILI_PDL=0 and 1: equal bits."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = []
    for pdl in "01":
        path = str(tmp_path / pdl)
        subprocess.run([sys.executable, "-c", CHAIN, root, path], check=True, timeout=300,
                       env=dict(os.environ, AKILI_PDL=pdl))
        got.append(torch.load(path))
    assert len(got[0]) == 24 and all(torch.equal(a, b) for a, b in zip(*got))
    assert got[0][21].tolist() == [90, 80] and not any(torch.isnan(t.float()).any() for t in got[0])
