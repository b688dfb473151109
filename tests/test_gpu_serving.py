"""The serving operators on the GPU against their fp64 statements
(serving_reference.py holds the definitions and the derived error bounds)."""
import itertools
import math

import pytest

torch = pytest.importorskip("torch")

from akili_bench_b200 import abi, ops  # noqa: E402
import serving_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def prefix(lens):
    return i32([0, *itertools.accumulate(lens)])


@pytest.fixture(autouse=True)
def clean_status():
    ops.device_status()
    yield
    assert ops.device_status() == 0


def took_bad_index():
    return ops.device_status() == abi.STATUS_BAD_INDEX


# -------------------------------------------------------------------- rope --
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("tokens,hq,hk,d,rot", [(1, 1, 1, 8, 8), (5, 4, 2, 64, 64), (33, 7, 1, 96, 64), (2, 32, 8, 128, 128),
                                               (300, 3, 3, 80, 20), (3, 2, 0, 10, 6), (4, 0, 5, 256, 32),
                                               (700, 32, 8, 128, 128), (3, 2, 1, 1040, 640)])
@pytest.mark.parametrize("interleaved,inverse", [(False, False), (True, False), (False, True), (True, True)])
def test_rope(dtype, tokens, hq, hk, d, rot, interleaved, inverse):
    g = gen(tokens * 131 + d)
    q, k = normal(g, (tokens, hq, d), dtype), normal(g, (tokens, hk, d), dtype)
    pos = torch.randint(0, 500, (tokens,), generator=g, dtype=torch.int32)
    table = normal(g, (500, rot), F32)
    got = ops.rope(q.cuda(), k.cuda(), pos.cuda(), table.cuda(), interleaved=interleaved, inverse=inverse)
    for name, x, y in zip("qk", (q, k), got):
        want, bound = ref.rotate(x, pos, table, interleaved, inverse)
        ref.assert_within(y, want, bound, name)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_strided_views_and_in_place(dtype, interleaved):
    """q and k as views of one projection's output, rotated in place; the bytes around them stay."""
    g = gen(5)
    fused = normal(g, (19, (6 + 2 + 2) * 64 + 16), dtype).cuda()
    before = fused.clone()
    q, k = fused[:, 16:16 + 384].view(19, 6, 64), fused[:, 400:528].view(19, 2, 64)
    pos = torch.arange(19, dtype=torch.int32) * 7 % 100
    table = normal(g, (100, 32), F32)
    want = [ref.rotate(x.cpu().clone(), pos, table, interleaved) for x in (q, k)]
    ops.rope(q, k, pos.cuda(), table.cuda(), interleaved=interleaved, q_out=q, k_out=k)
    for x, (y, b) in zip((q, k), want):
        ref.assert_within(x, y, b)
    assert torch.equal(fused[:, :16], before[:, :16]) and torch.equal(fused[:, 528:], before[:, 528:])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("hq,hk,d,rot", [(4, 2, 64, 64), (5, 0, 80, 48), (1, 1, 128, 32), (3, 2, 24, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_of_many_tokens(dtype, hq, hk, d, rot, interleaved):
    """Enough tokens for the whole-row form; rows of a wider buffer, one position outside the table."""
    g = gen(hq * d)
    t = 3700
    fused = normal(g, (t, (hq + hk) * d + 16), dtype)
    q, k = fused[:, :hq * d].view(t, hq, d), fused[:, hq * d:(hq + hk) * d].view(t, hk, d)
    pos = torch.randint(0, 900, (t,), generator=g, dtype=torch.int32)
    pos[1234] = 900
    table = normal(g, (900, rot), F32)
    dev = fused.cuda()
    dq, dk = dev[:, :hq * d].view(t, hq, d), dev[:, hq * d:(hq + hk) * d].view(t, hk, d)
    out_q, out_k = torch.full_like(dq, 3.0).contiguous(), torch.full_like(dk, 3.0).contiguous()
    for inverse in (False, True):
        ops.rope(dq, dk, pos.cuda(), table.cuda(), interleaved=interleaved, inverse=inverse, q_out=out_q, k_out=out_k)
        assert took_bad_index()
        on = pos < 900
        for x, y in ((q, out_q), (k, out_k)):
            want, bound = ref.rotate(x[on], pos[on], table, interleaved, inverse)
            ref.assert_within(y.cpu()[on], want, bound)
            assert (y[1234] == 3.0).all()
    ops.rope(dq, dk, pos.cuda(), table.cuda(), interleaved=interleaved, q_out=dq, k_out=dk)
    assert took_bad_index()
    want, bound = ref.rotate(q[on], pos[on], table, interleaved)
    ref.assert_within(dq.cpu()[on], want, bound)
    assert torch.equal(dev[:, (hq + hk) * d:].cpu(), fused[:, (hq + hk) * d:])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads_first", [False, True])
def test_rope_append_of_many_tokens(dtype, heads_first):
    g = gen(91)
    t, hq, hk, d, page = 3800, 3, 2, 64, 24
    q, k, v = (normal(g, (t, h, d), dtype) for h in (hq, hk, hk))
    pages = t // page + 5
    shape = (pages, hk, page, d) if heads_first else (pages, page, hk, d)
    kp, vp = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    if heads_first:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    slots = torch.randperm(pages * page, generator=g)[:t]
    slots[7], slots[3000] = -1, pages * page
    pos = torch.randint(0, 200, (t,), generator=g, dtype=torch.int32)
    table = normal(g, (200, d), F32)
    k_out = torch.empty(hk, t, d, dtype=dtype, device="cuda").transpose(0, 1)
    out = ops.rope_append(q.cuda(), k.cuda(), v.cuda(), pos.cuda(), table.cuda(), slots.cuda(), kp, vp, k_out=k_out)
    assert took_bad_index()
    ref.assert_within(out, *ref.rotate(q, pos, table))
    want, bound = ref.rotate(k, pos, table)
    ref.assert_within(k_out, want, bound)
    on = (slots >= 0) & (slots < pages * page)
    kf, vf = kp.cpu().reshape(-1, hk, d), vp.cpu().reshape(-1, hk, d)
    ref.assert_within(kf[slots[on]], want[on], bound[on])
    assert torch.equal(vf[slots[on]], v[on])
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots[on]] = False
    assert torch.isnan(kf[rest]).all() and torch.isnan(vf[rest]).all()


def test_rope_unaligned_view_takes_the_elementwise_form():
    g = gen(6)
    buf = normal(g, (9 * 4 * 64 + 1,), F16).cuda()
    q = buf[1:].view(9, 4, 64)
    pos, table = torch.arange(9, dtype=torch.int32), normal(g, (9, 64), F32)
    out, _ = ops.rope(q, q, pos.cuda(), table.cuda())
    want, bound = ref.rotate(q.cpu(), pos, table)
    ref.assert_within(out, want, bound)


def test_rope_inverse_is_the_gradient():
    """<g, R x> against central differences of x, and R^T g = inverse(g), in fp32."""
    g = gen(7)
    x, w = normal(g, (4, 3, 32), F32), normal(g, (4, 3, 32), F32)
    pos = i32([3, 0, 77, 41])
    table = ops.rope_table(100, 32)
    none = torch.empty(4, 0, 32, device="cuda")
    for interleaved in (False, True):
        grad = ops.rope(w.cuda(), none, pos.cuda(), table, interleaved=interleaved, inverse=True)[0].double().cpu()
        want, bound = ref.rotate(w, pos, table.cpu(), interleaved, inverse=True)
        ref.assert_within(grad, want, bound)
        h = 2.0 ** -4  # the map is linear: differences have no truncation error, only fp32 rounding
        for at in [(0, 0, 0), (2, 1, 5), (3, 2, 31), (2, 0, 17)]:
            up, down = x.clone(), x.clone()
            up[at] += h
            down[at] -= h
            f = [(ops.rope(z.cuda(), none, pos.cuda(), table, interleaved=interleaved)[0].double().cpu() *
                  w.double()).sum() for z in (up, down)]
            # each of the 96 terms is rounded to 2^-24 of at most |w| (|x1| + |x2|) <= 50
            assert abs((f[0] - f[1]) / (2 * h) - grad[at]) <= 2 * 96 * 50 * 2.0 ** -23 / (2 * h)


def test_rope_skips_positions_outside_the_table():
    g = gen(8)
    q = normal(g, (4, 2, 16), F16).cuda()
    out = torch.full_like(q, 7.0)
    pos, table = i32([0, -1, 9, 10]), normal(g, (10, 16), F32)
    ops.rope(q, q[:, :0], pos.cuda(), table.cuda(), q_out=out)
    assert took_bad_index()
    want, bound = ref.rotate(q.cpu()[[0, 2]], pos[[0, 2]], table)
    ref.assert_within(out[[0, 2]], want, bound)
    assert (out[[1, 3]] == 7.0).all()


def frequencies(rot, base, scaling, factor, orig, low, high):
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "base":
        b = base * factor ** (rot / (rot - 2.0))
        f = [b ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "bands":
        out = []
        for x in f:
            wave = 2 * math.pi / x
            if wave < orig / high:
                out.append(x)
            elif wave > orig / low:
                out.append(x / factor)
            else:
                t = (orig / wave - low) / (high - low)
                out.append((1 - t) * x / factor + t * x)
        f = out
    if scaling == "ramp":
        at = lambda turns: rot * math.log(orig / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(high)), 0), min(math.ceil(at(low)), rot - 1)
        f = [(x / factor) * r + x * (1 - r)
             for x, r in ((x, min(max((i - lo) / (hi - lo), 0.0), 1.0)) for i, x in enumerate(f))]
    return torch.tensor(f, dtype=torch.float64)


@pytest.mark.parametrize("rot", [2, 64, 128])
@pytest.mark.parametrize("scaling,factor,orig,low,high,amp", [
    (None, 1.0, 0, 0, 0, 1.0), (None, 1.0, 0, 0, 0, 0.5), ("linear", 4.0, 0, 0, 0, 0.0), ("base", 8.0, 0, 0, 0, 0.0),
    ("bands", 8.0, 8192, 1.0, 4.0, 0.0), ("ramp", 16.0, 4096, 1.0, 32.0, 0.0), ("ramp", 2.0, 2048, 1.0, 32.0, 1.0)])
def test_rope_table(rot, scaling, factor, orig, low, high, amp):
    if scaling == "base" and rot == 2:
        pytest.skip("base scaling needs rot_dim > 2")
    n = 131072 if rot == 64 else 5000
    got = ops.rope_table(n, rot, 10000.0, scaling, factor, orig, low, high, amp).double().cpu()
    a = torch.arange(n, dtype=torch.float64)[:, None] * frequencies(rot, 10000.0, scaling, factor, orig, low, high)
    size = amp or (0.1 * math.log(factor) + 1 if scaling == "ramp" else 1.0)
    want = torch.cat([size * a.cos(), size * a.sin()], 1)
    # fp32 rounding, and 2^-50 relative of the angle for the frequencies' and the product's fp64 rounding
    assert ((got - want).abs() <= 2.0 ** -24 * size * 1.001 + size * n * 2.0 ** -50).all()


# ----------------------------------------------------------------- append --
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,d,rot,page", [(1, 2, 1, 8, 8, 8), (37, 8, 2, 128, 128, 16), (50, 3, 3, 80, 40, 24),
                                                    (20, 4, 4, 12, 6, 5)])
def test_rope_append(dtype, heads_first, tokens, hq, hk, d, rot, page):
    g = gen(tokens + d)
    q, k, v = (normal(g, (tokens, h, d), dtype) for h in (hq, hk, hk))
    pages = tokens // page + 3
    shape = (pages, hk, page, d) if heads_first else (pages, page, hk, d)
    kp, vp = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    if heads_first:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    if tokens > 3:
        slots[2] = -1
    pos = torch.randint(0, 200, (tokens,), generator=g, dtype=torch.int32)
    table = normal(g, (200, rot), F32)
    for interleaved in (False, True):
        out = ops.rope_append(q.cuda(), k.cuda(), v.cuda(), pos.cuda(), table.cuda(), slots.cuda(), kp, vp,
                              interleaved=interleaved)
        ref.assert_within(out, *ref.rotate(q, pos, table, interleaved))
        want, bound = ref.rotate(k, pos, table, interleaved)
        kf, vf = kp.cpu().reshape(-1, hk, d), vp.cpu().reshape(-1, hk, d)
        on = slots >= 0
        ref.assert_within(kf[slots[on]], want[on], bound[on])
        assert torch.equal(vf[slots[on]], v[on])
        rest = torch.ones(pages * page, dtype=torch.bool)
        rest[slots[on]] = False
        assert torch.isnan(kf[rest]).all() and torch.isnan(vf[rest]).all()


@pytest.mark.parametrize("in_place", [False, True])
def test_rope_append_keeps_the_rotated_keys_of_every_token(in_place):
    g = gen(77)
    q, k, v = (normal(g, (21, h, 64), BF16) for h in (4, 2, 2))
    pages = torch.zeros(2, 16, 2, 64, dtype=BF16, device="cuda")
    v_pages = torch.zeros_like(pages)
    slots = torch.arange(21)
    slots[5] = -1  # padding goes to no page, but is rotated
    pos, table = torch.arange(21, dtype=torch.int32), normal(g, (30, 64), F32)
    dev_k = k.cuda()
    k_out = dev_k if in_place else torch.empty(2, 21, 64, dtype=BF16, device="cuda").transpose(0, 1)
    ops.rope_append(q.cuda(), dev_k, v.cuda(), pos.cuda(), table.cuda(), slots.cuda(), pages, v_pages, k_out=k_out)
    want, bound = ref.rotate(k, pos, table)
    ref.assert_within(k_out, want, bound)
    on = slots >= 0
    flat = pages.view(-1, 2, 64)
    assert torch.equal(flat[slots[on].cuda()], k_out[on.cuda()])
    assert (flat[5] == 0).all() and (v_pages.view(-1, 2, 64)[5] == 0).all()


def test_rope_append_skips_slots_outside_the_pages():
    q = torch.ones(2, 1, 8, dtype=F16, device="cuda")
    pages = torch.zeros(2, 4, 1, 8, dtype=F16, device="cuda")
    ops.rope_append(q, q, q, i32([0, 0]).cuda(), ops.rope_table(1, 8), torch.tensor([8, -2], device="cuda"), pages[:2],
                    pages[:2].clone())
    assert took_bad_index()
    assert (pages == 0).all()


# ----------------------------------------------------------------- prompts --
PROMPTS = [
    # (query lengths, key lengths or None, hq, hk, d)
    ([1], None, 1, 1, 8),
    ([128], None, 2, 2, 64),
    ([129, 1, 0, 300], None, 4, 2, 128),
    ([257], None, 1, 1, 128),
    ([33, 7, 64, 255, 256, 1], None, 8, 1, 64),
    ([100, 90], None, 7, 1, 80),
    ([5, 130, 0, 20], [300, 130, 17, 0], 6, 2, 96),
    ([200, 40], [70, 41], 3, 3, 128),      # more queries than keys: the first rows see nothing
    ([3] * 70, None, 4, 4, 16),
    ([700, 513], None, 2, 1, 128),
    ([31, 65], [1000, 65], 16, 2, 120),
    ([1, 2], None, 72, 1, 64),
    ([5, 70], None, 131, 1, 64),           # a group that no divisor packs
]


def check_prompt(q, k, v, qlens, klens, causal, got, lse=None, scale=None):
    at = ak = 0
    for b, (n, m) in enumerate(zip(qlens, klens)):
        seen = ref.causal(n, m) if causal else torch.ones(n, m, dtype=torch.bool)
        o, l, bound, l_bound = ref.attend(q[at:at + n], k[ak:ak + m], v[ak:ak + m], seen, scale)
        ref.assert_within(got[at:at + n], o, bound, f"sequence {b}")
        if lse is not None:
            ref.assert_within(lse[at:at + n], l, l_bound, f"lse of sequence {b}")
        at, ak = at + n, ak + m


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_prompt_attention(dtype, causal, case):
    qlens, klens, hq, hk, d = PROMPTS[case]
    klens = klens or qlens
    g = gen(case)
    q, k, v = normal(g, (sum(qlens), hq, d), dtype), normal(g, (sum(klens), hk, d), dtype), \
        normal(g, (sum(klens), hk, d), dtype)
    got, lse = ops.prompt_attention(q.cuda(), k.cuda(), v.cuda(), prefix(qlens).cuda(), prefix(klens).cuda(),
                                    causal=causal, return_lse=True)
    check_prompt(q, k, v, qlens, klens, causal, got, lse)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,hk,d", [(16, 8, 128), (16, 16, 64), (28, 4, 80), (48, 48, 128)])
def test_prompt_attention_with_more_tiles_than_sms(dtype, causal, hq, hk, d):
    """Two tiles a CTA, blocks taken over from the rest of the grid (small batches have one tile a CTA)."""
    g = gen(hq + d)
    qlens, klens = [420, 1, 0, 333, 130, 64], [500, 33, 7, 333, 129, 64]
    q, k, v = normal(g, (sum(qlens), hq, d), dtype), normal(g, (sum(klens), hk, d), dtype), \
        normal(g, (sum(klens), hk, d), dtype)
    got, lse = ops.prompt_attention(q.cuda(), k.cuda(), v.cuda(), prefix(qlens).cuda(), prefix(klens).cuda(),
                                    causal=causal, return_lse=True)
    check_prompt(q, k, v, qlens, klens, causal, got, lse)


def test_prompt_attention_without_any_key():
    q = torch.ones(130, 4, 64, dtype=F16, device="cuda")
    none = torch.empty(0, 2, 64, dtype=F16, device="cuda")
    for causal in (True, False):
        got, lse = ops.prompt_attention(q, none, none, i32([0, 100, 130]).cuda(), i32([0, 0, 0]).cuda(), causal=causal,
                                        return_lse=True)
        assert (got == 0).all() and (lse == -math.inf).all()


def test_attention_refuses_broadcast_strides():
    """An expanded axis has stride 0, which the tile loads cannot address."""
    q = torch.ones(8, 4, 64, dtype=F16, device="cuda")
    k = torch.ones(8, 1, 64, dtype=F16, device="cuda").expand(8, 4, 64)
    with pytest.raises(abi.AkiliError) as e:
        ops.prompt_attention(q, k, q, i32([0, 8]).cuda())
    assert e.value.code == abi.E_SHAPE
    pages = torch.ones(1, 8, 1, 64, dtype=F16, device="cuda").expand(2, 8, 2, 64)
    with pytest.raises(abi.AkiliError) as e:
        ops.tree_attention(q, pages, pages, i32([[0, 1]]).cuda(), i32([8]).cuda(), i32([0, 8]).cuda())
    assert e.value.code == abi.E_SHAPE


def test_prompt_attention_large_scores_and_scale():
    """Rising scores (the running maximum moves in every block) and scores in the hundreds."""
    g = gen(3)
    n, d = 600, 64
    q = normal(g, (n, 2, d), F16).abs()
    k = normal(g, (n, 2, d), F16).abs() * (torch.arange(n)[:, None, None] / 60.0).half()
    v = normal(g, (n, 2, d), F16)
    for scale in (None, 1.0, 0.01):
        got = ops.prompt_attention(q.cuda(), k.cuda(), v.cuda(), i32([0, n]).cuda(), softmax_scale=scale)
        check_prompt(q, k, v, [n], [n], True, got, scale=scale)
        back = ops.prompt_attention(q.cuda(), k.flip(0).cuda(), v.cuda(), i32([0, n]).cuda(), softmax_scale=scale)
        check_prompt(q, k.flip(0), v, [n], [n], True, back, scale=scale)


def test_prompt_attention_strided_views():
    """q, k, v as views of one projection; output into a head-major buffer."""
    g = gen(4)
    qlens, hq, hk, d = [150, 3, 260], 6, 2, 64
    t = sum(qlens)
    fused = normal(g, (t, (hq + 2 * hk) * d + 8), BF16)
    dev = fused.cuda()
    parts = lambda x: (x[:, 8:8 + hq * d].view(t, hq, d), x[:, 8 + hq * d:8 + (hq + hk) * d].view(t, hk, d),  # noqa: E731
                       x[:, 8 + (hq + hk) * d:].view(t, hk, d))
    out = torch.full((hq, t, d), float("nan"), dtype=BF16, device="cuda")
    ops.prompt_attention(*parts(dev), prefix(qlens).cuda(), out=out.transpose(0, 1))
    check_prompt(*parts(fused), qlens, qlens, True, out.transpose(0, 1))


def test_prompt_attention_other_sequences_do_not_leak():
    """A sequence full of NaN and infinities leaves its neighbours as they are."""
    g = gen(9)
    qlens, hq, hk, d = [70, 150, 90], 4, 2, 128
    q, k, v = (normal(g, (sum(qlens), h, d), F16) for h in (hq, hk, hk))
    for x in (q, k, v):
        x[70:150] = float("nan")
        x[150:220] = float("inf")
    for causal in (True, False):
        got = ops.prompt_attention(q.cuda(), k.cuda(), v.cuda(), prefix(qlens).cuda(), causal=causal).cpu()
        for a, n in ((0, 70), (220, 90)):
            seen = ref.causal(n, n) if causal else torch.ones(n, n, dtype=torch.bool)
            o, _, bound, _ = ref.attend(q[a:a + n], k[a:a + n], v[a:a + n], seen)
            ref.assert_within(got[a:a + n], o, bound)


def test_prompt_attention_masked_keys_may_be_nan():
    """Keys after a query are not seen, whatever they hold (their values are finite)."""
    g = gen(10)
    n, d = 300, 64
    q, k, v = (normal(g, (n, 1, d), BF16) for _ in range(3))
    k[200:] = float("nan")
    got = ops.prompt_attention(q.cuda(), k.cuda(), v.cuda(), i32([0, n]).cuda()).cpu()
    o, _, bound, _ = ref.attend(q[:200], k[:200], v[:200], ref.causal(200, 200))
    ref.assert_within(got[:200], o, bound)
    assert torch.isnan(got[200:]).all()


def test_prompt_attention_rows_outside_the_sequences_are_not_written():
    g = gen(11)
    q = normal(g, (50, 2, 64), F16).cuda()
    out = torch.full_like(q, 5.0)
    ops.prompt_attention(q, q, q, i32([0, 20, 33]).cuda(), out=out)
    assert (out[33:] == 5.0).all()
    check_prompt(q.cpu(), q.cpu(), q.cpu(), [20, 13], [20, 13], True, out[:33])


def test_prompt_attention_lengths_past_the_buffers_are_clamped():
    g = gen(12)
    q = normal(g, (40, 2, 64), F16).cuda()
    got = ops.prompt_attention(q, q, q, i32([0, 64]).cuda())
    check_prompt(q.cpu(), q.cpu(), q.cpu(), [40], [40], True, got)


# ------------------------------------------------------------------- trees --
def make_cache(g, lens, page, hk, d, dtype, heads_first=False, extra=2):
    """NaN-filled pages, a shuffled page table with -1 past each sequence, and a writer of entries."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + extra
    shape = (total, hk, page, d) if heads_first else (total, page, hk, d)
    kp, vp = (torch.full(shape, float("nan"), dtype=dtype) for _ in range(2))
    order = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    at, ks, vs = 0, [], []
    for b, n in enumerate(lens):
        ids = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = i32(ids)
        k, v = normal(g, (n, hk, d), dtype), normal(g, (n, hk, d), dtype)
        ks.append(k)
        vs.append(v)
        for j in range(n):
            for pages, x in ((kp, k), (vp, v)):
                if heads_first:
                    pages[ids[j // page], :, j % page] = x[j]
                else:
                    pages[ids[j // page], j % page] = x[j]
    kd, vd = kp.cuda(), vp.cuda()
    if heads_first:
        kd, vd = kd.transpose(1, 2), vd.transpose(1, 2)
    return kd, vd, table, ks, vs


def random_parents(g, n, roots=1):
    return [-1 if i < roots else int(torch.randint(max(0, i - 6), i, (1,), generator=g)) for i in range(n)]


TREES = [
    # (contexts, new tokens, page, hq, hk, d, heads_first, tree)
    ([0], [1], 8, 1, 1, 8, False, False),
    ([1], [1], 16, 4, 4, 64, False, False),
    ([127, 128, 129], [1, 1, 1], 16, 8, 2, 128, False, False),
    ([1000, 3, 0, 515], [1, 1, 1, 1], 24, 7, 1, 80, True, False),
    ([2500], [1], 64, 32, 32, 128, False, False),
    ([40, 300], [130, 57], 32, 4, 1, 64, False, False),       # chunks of prompts
    ([70, 0, 513, 20], [16, 5, 33, 0], 16, 8, 2, 128, False, True),
    ([640], [64], 128, 32, 8, 128, True, True),
    ([100, 1], [100, 129], 8, 4, 2, 96, False, True),
    ([33] * 40, [3] * 40, 16, 6, 2, 64, False, True),
    ([4000, 17], [40, 64], 256, 8, 1, 128, False, True),
    ([90], [300], 40, 2, 1, 128, False, True),
    ([1500] * 3, [1] * 3, 16, 64, 1, 128, False, False),
    ([300, 9], [1, 2], 16, 131, 1, 64, False, False),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", range(len(TREES)))
def test_tree_attention(dtype, case):
    ctx, new, page, hq, hk, d, heads_first, tree = TREES[case]
    g = gen(100 + case)
    kp, vp, table, ks, vs = make_cache(g, [c + n for c, n in zip(ctx, new)], page, hk, d, dtype, heads_first)
    q = normal(g, (sum(new), hq, d), dtype)
    parents = [random_parents(g, n, roots=1 + b % 2) for b, n in enumerate(new)]
    cu = prefix(new).cuda()
    mask = None
    if tree:
        mask = ops.tree_mask(i32(sum(parents, [])).cuda(), cu, max(new))
    got, lse = ops.tree_attention(q.cuda(), kp, vp, table.cuda(), i32(ctx).cuda(), cu, mask, return_lse=True)
    at = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        seen = ref.tree_seen(c, parents[b]) if tree else ref.causal(n, c + n)
        o, l, bound, l_bound = ref.attend(q[at:at + n], ks[b], vs[b], seen)
        ref.assert_within(got[at:at + n], o, bound, f"sequence {b}")
        ref.assert_within(lse[at:at + n], l, l_bound, f"lse of sequence {b}")
        at += n


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk,new", [(5, 1, 3), (16, 1, 1), (4, 2, 11), (8, 2, 13), (3, 1, 40), (8, 2, 50), (16, 2, 33)])
def test_tree_attention_row_forms_and_rising_scores(dtype, d, hq, hk, new):
    """Every row form (16 to 256 rows of an item), scores that rise along the context (the running maximum
    moves in most blocks) or fall, contexts that are cut between CTAs and ones that are not."""
    g = gen(hq * 100 + new)
    ctx = [2500, 0, 260, 77]
    for tree, rise in ((True, True), (False, True), (True, False)):
        kp, vp, table, ks, vs = make_cache(g, [c + new for c in ctx], 16, hk, d, dtype)
        for b, c in enumerate(ctx):  # scale entry j's key by its place
            f = (torch.arange(c + new) + 1.0) / 40.0
            f = (f if rise else f.flip(0))[:, None, None]
            ks[b] = (ks[b].abs() * f).to(dtype)
            for j in range(c + new):
                kp[int(table[b, j // 16]), j % 16] = ks[b][j].cuda()
        q = normal(g, (4 * new, hq, d), dtype).abs()
        parents = [random_parents(g, new) for _ in ctx]
        cu = prefix([new] * 4).cuda()
        mask = ops.tree_mask(i32(sum(parents, [])).cuda(), cu, new) if tree else None
        got, lse = ops.tree_attention(q.cuda(), kp, vp, table.cuda(), i32(ctx).cuda(), cu, mask, softmax_scale=0.02,
                                      return_lse=True)
        for b, c in enumerate(ctx):
            seen = ref.tree_seen(c, parents[b]) if tree else ref.causal(new, c + new)
            o, l, bound, l_bound = ref.attend(q[b * new:(b + 1) * new], ks[b], vs[b], seen, 0.02)
            ref.assert_within(got[b * new:(b + 1) * new], o, bound, f"sequence {b}")
            ref.assert_within(lse[b * new:(b + 1) * new], l, l_bound, f"lse of sequence {b}")


def test_tree_mask_bits():
    g = gen(20)
    new = [1, 40, 0, 97, 32]
    parents = [random_parents(g, n, roots=2) for n in new]
    got = ops.tree_mask(i32(sum(parents, [])).cuda(), prefix(new).cuda(), max(new)).cpu()
    want = torch.cat([ref.bits_of(ref.tree_seen(0, p), 4) for p in parents])
    assert torch.equal(got, want)


def test_tree_mask_records_bad_parents():
    got = ops.tree_mask(i32([-1, 1, -5, 0]).cuda(), i32([0, 4]).cuda(), 4).cpu()
    assert took_bad_index()
    assert got.tolist() == [[1], [2], [4], [9]]
    ops.tree_mask(i32([-1] * 40).cuda(), i32([0, 40]).cuda(), 32)
    assert took_bad_index()


def test_tree_attention_rows_that_see_nothing():
    """No context and an empty mask row: 0 and lse -inf, also next to rows that see something."""
    g = gen(21)
    kp, vp, table, ks, vs = make_cache(g, [6, 140], 8, 2, 64, F16)
    q = normal(g, (6 + 4, 4, 64), F16)
    seen = [torch.eye(6, dtype=torch.bool), torch.zeros(4, 4, dtype=torch.bool)]
    seen[0][[1, 4]] = False
    mask = torch.cat([ref.bits_of(s, 1) for s in seen])
    got, lse = ops.tree_attention(q.cuda(), kp, vp, table.cuda(), i32([0, 136]).cuda(), i32([0, 6, 10]).cuda(),
                                  mask.cuda(), return_lse=True)
    at = 0
    for b, (c, s) in enumerate(zip([0, 136], seen)):
        n = s.shape[0]
        full = torch.cat([torch.ones(n, c, dtype=torch.bool), s], 1)
        o, l, bound, l_bound = ref.attend(q[at:at + n], ks[b], vs[b], full)
        ref.assert_within(got[at:at + n], o, bound)
        ref.assert_within(lse[at:at + n], l, l_bound)
        at += n
    assert (got[[1, 4]] == 0).all() and (lse[[1, 4]] == -math.inf).all()


def test_tree_attention_layers_view_workspace_and_repeat():
    """Pages of one layer of a larger buffer, a caller's workspace, bitwise equal repeats."""
    g = gen(22)
    ctx, new, page, hq, hk, d = [900, 77], [5, 9], 16, 8, 2, 128
    kp, vp, table, ks, vs = make_cache(g, [c + n for c, n in zip(ctx, new)], page, hk, d, BF16)
    both = torch.full((2, 3, *kp.shape), float("nan"), dtype=BF16, device="cuda")
    both[0, 1], both[1, 1] = kp, vp
    q = normal(g, (14, hq, d), BF16).cuda()
    args = (q, both[0, 1], both[1, 1], table.cuda(), i32(ctx).cuda(), i32([0, 5, 14]).cuda())
    first = ops.tree_attention(*args)
    n = ops.tree_attention_workspace(q, both[0, 1], args[3], args[4])
    ws = torch.full((max(n, 1),), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(ops.tree_attention(*args, workspace=ws), first)
    assert torch.equal(ops.tree_attention(*args), first)
    at = 0
    for b, (c, m) in enumerate(zip(ctx, new)):
        o, _, bound, _ = ref.attend(q[at:at + m].cpu(), ks[b], vs[b], ref.causal(m, c + m))
        ref.assert_within(first[at:at + m], o, bound)
        at += m


def test_tree_attention_workspace_must_be_large_enough():
    g = gen(26)
    kp, vp, table, _, _ = make_cache(g, [40], 8, 1, 64, F16)
    q = normal(g, (1, 2, 64), F16).cuda()
    args = (q, kp, vp, table.cuda(), i32([39]).cuda(), i32([0, 1]).cuda())
    n = ops.tree_attention_workspace(q, kp, args[3], args[4])
    for size, code in ((n - 1, abi.E_WORKSPACE), (n, abi.OK)):
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        if code == abi.OK:
            ops.tree_attention(*args, workspace=ws)
        else:
            with pytest.raises(abi.AkiliError) as e:
                ops.tree_attention(*args, workspace=ws)
            assert e.value.code == code


def test_tree_attention_invalid_pages_read_as_zeros():
    g = gen(23)
    kp, vp, table, ks, vs = make_cache(g, [65], 16, 1, 64, F16)
    q = normal(g, (1, 2, 64), F16)
    table[0, 1], table[0, 3] = -7, 1 << 20
    got = ops.tree_attention(q.cuda(), kp, vp, table.cuda(), i32([64]).cuda(), i32([0, 1]).cuda())
    assert took_bad_index()
    for x in (ks[0], vs[0]):
        x[16:32] = 0
        x[48:64] = 0
    o, _, bound, _ = ref.attend(q, ks[0], vs[0], ref.causal(1, 65))
    ref.assert_within(got, o, bound)


def test_tree_attention_contexts_past_the_table_are_clamped():
    g = gen(24)
    kp, vp, table, ks, vs = make_cache(g, [48], 16, 1, 64, F16)
    q = normal(g, (1, 1, 64), F16)
    got = ops.tree_attention(q.cuda(), kp, vp, table.cuda(), i32([1 << 20]).cuda(), i32([0, 1]).cuda())
    assert took_bad_index()
    o, _, bound, _ = ref.attend(q, ks[0], vs[0], torch.ones(1, 48, dtype=torch.bool))
    ref.assert_within(got, o, bound)


def test_offsets_past_32_bits():
    """Cache entries more than 2^32 elements into their buffer."""
    g = gen(25)
    hk, d, page = 8, 128, 128
    per = page * hk * d
    pages = (1 << 32) // per + 4
    kp, vp = (torch.empty(pages, page, hk, d, dtype=F16, device="cuda") for _ in range(2))
    ids = [pages - 1, 0, pages - 2]
    k, v = normal(g, (300, hk, d), F16), normal(g, (300, hk, d), F16)
    slots = torch.tensor([ids[j // page] * page + j % page for j in range(300)])
    pos, table = torch.zeros(300, dtype=torch.int32), torch.tensor([[1.0] * 64 + [0.0] * 64])
    q = normal(g, (300, hk, d), F16)
    ops.rope_append(q.cuda(), k.cuda(), v.cuda(), pos.cuda(), table.cuda(), slots.cuda(), kp, vp)
    got = ops.tree_attention(q[299:].cuda(), kp, vp, i32([ids]).cuda(), i32([299]).cuda(), i32([0, 1]).cuda())
    o, _, bound, _ = ref.attend(q[299:], k, v, ref.causal(1, 300))
    ref.assert_within(got, o, bound)
    lens = ops.cache_accept(kp, vp, i32([ids]).cuda(), i32([290]).cuda(), i32([[2, 7]]).cuda(), i32([2]).cuda())
    assert lens.tolist() == [292]
    assert torch.equal(kp.flatten(0, 1)[slots[290:292].cuda()].cpu(), k[[292, 297]])
    assert torch.equal(vp.flatten(0, 1)[slots[290:292].cuda()].cpu(), v[[292, 297]])


# ------------------------------------------------------------------ accept --
@pytest.mark.parametrize("dtype,hk,d", [(F16, 8, 128), (BF16, 1, 8), (F32, 3, 20), (torch.float8_e4m3fn, 2, 64), (F16, 3, 5)])
@pytest.mark.parametrize("heads_first", [False, True])
def test_cache_accept(dtype, hk, d, heads_first):
    g = gen(hk * d)
    ctx, new, page, layers = [0, 30, 7, 100, 55], [64, 20, 200, 1, 9], 12, 3
    took = [64, 5, 150, 1, 0]
    need = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    pages = sum(need) + 1
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((5, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = i32(order[at:at + n])
        at += n
    shape = (layers, pages, hk, page, d) if heads_first else (layers, pages, page, hk, d)
    kp, vp = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    if heads_first:
        kp, vp = kp.transpose(2, 3), vp.transpose(2, 3)
    acc = torch.full((5, 160), -9, dtype=torch.int32)
    for b, (n, a) in enumerate(zip(new, took)):
        acc[b, :a] = torch.randperm(n, generator=g)[:a].sort().values.int()
    if dtype == torch.float8_e4m3fn:
        want_k, want_v = kp.clone().view(torch.uint8), vp.clone().view(torch.uint8)
    else:
        want_k, want_v = kp.clone(), vp.clone()
    old_k, old_v = want_k.clone(), want_v.clone()
    for b, a in enumerate(took):
        for i in range(a):
            s, t = ctx[b] + int(acc[b, i]), ctx[b] + i
            want_k[:, table[b, t // page], t % page] = old_k[:, table[b, s // page], s % page]
            want_v[:, table[b, t // page], t % page] = old_v[:, table[b, s // page], s % page]
    kd, vd = kp.cuda(), vp.cuda()
    if dtype == torch.float8_e4m3fn:
        kd, vd = kd.view(torch.uint8), vd.view(torch.uint8)
    lens = ops.cache_accept(kd, vd, table.cuda(), i32(ctx).cuda(), acc.cuda(), i32(took).cuda())
    assert lens.tolist() == [c + a for c, a in zip(ctx, took)]
    assert torch.equal(kd.cpu(), want_k) and torch.equal(vd.cpu(), want_v)


def test_cache_accept_skips_what_is_out_of_range():
    kp = torch.arange(4 * 8, dtype=F32).view(4, 8, 1, 1).cuda()
    vp = kp.clone()
    table = i32([[2, 9]])
    # 3 -> 0 moves; 3 again does not ascend; 9 lies in a page that is not there; 40 past the table
    lens = ops.cache_accept(kp, vp, table.cuda(), i32([1]).cuda(), i32([[3, 3, 9, 40]]).cuda(), i32([4]).cuda())
    assert took_bad_index()
    want = torch.arange(4 * 8, dtype=F32).view(4, 8)
    want[2, 1] = want[2, 4].clone()
    assert torch.equal(kp.view(4, 8).cpu(), want) and torch.equal(vp, kp)
    assert lens.tolist() == [5]


# ------------------------------------------------------- streams and graphs --
def test_another_stream_and_graph_capture():
    g = gen(30)
    ctx, page, hq, hk, d = [300, 41], 16, 8, 2, 64
    kp, vp, table, _, _ = make_cache(g, [c + 1 for c in ctx], page, hk, d, F16, extra=40)
    q = normal(g, (2, hq, d), F16).cuda()
    lens, cu, table = i32(ctx).cuda(), i32([0, 1, 2]).cuda(), table.cuda()
    want = ops.tree_attention(q, kp, vp, table, lens, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ops.tree_attention(q, kp, vp, table, lens, cu, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    pq = normal(g, (90, hq, d), F16).cuda()
    cu_p = i32([0, 30, 90]).cuda()
    want_p = ops.prompt_attention(pq, pq, pq, cu_p)
    out, out_p = torch.zeros_like(q), torch.zeros_like(pq)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.tree_attention(q, kp, vp, table, lens, cu, out=out)  # the scratch pool of this stream exists
        graph = torch.cuda.CUDAGraph()
        out.zero_()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            ops.tree_attention(q, kp, vp, table, lens, cu, out=out)
            ops.prompt_attention(pq, pq, pq, cu_p, out=out_p)
        graph.replay()
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(out_p, want_p)
    lens.copy_(i32([200, 40]))  # a replay reads the lengths anew
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.tree_attention(q, kp, vp, table, lens, cu))


def test_zero_tokens_are_a_no_op():
    e = lambda *s: torch.empty(s, dtype=F16, device="cuda")  # noqa: E731
    before = ops.launch_count()
    assert ops.prompt_attention(e(0, 4, 64), e(0, 2, 64), e(0, 2, 64), i32([0]).cuda()).shape == (0, 4, 64)
    assert ops.tree_attention(e(0, 4, 64), e(3, 8, 2, 64), e(3, 8, 2, 64), torch.empty(0, 1, dtype=torch.int32).cuda(),
                              torch.empty(0, dtype=torch.int32).cuda(), i32([0]).cuda()).shape == (0, 4, 64)
    ops.rope(e(0, 4, 64), e(0, 2, 64), torch.empty(0, dtype=torch.int32).cuda(), ops.rope_table(1, 64))
    assert ops.launch_count() == before + 1  # the table
