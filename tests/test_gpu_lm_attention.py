"""``prefix_attention`` against its formula in 64 bits: lengths of zero and one, keys that end inside a
tile, ragged appends, rows that see nothing, what hidden keys hold, strides and padding."""

from __future__ import annotations

import pytest
import torch

from oracle import lm_oracle as O
from tests import lm_bars as bars
from tests.gpu_helpers import say

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def make(news, lengths, prefix, hq, hk, dim, dtype, seed=0, capacity=None, sessions=None, sharp=2.0):
    """q, caches, prefix and index tensors; what no query may see holds NaN."""
    g = torch.Generator().manual_seed(seed + 131 * prefix + sum(lengths))
    b = len(lengths)
    sessions = sessions or b + 2
    capacity = capacity or max(max(lengths), 1) + 5

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype)

    q = rand(sum(news), hq, dim, scale=sharp)
    k, v = rand(sessions, capacity, hk, dim), rand(sessions, capacity, hk, dim)
    slots = torch.randperm(sessions, generator=g)[:b].tolist()
    unused = [s for s in range(sessions) if s not in slots]
    for t in (k, v):
        for s in unused:
            t[s] = float("nan")
        for s, n in zip(slots, lengths):
            t[s, max(n, 0):] = float("nan")
    pk, pv = rand(prefix, hk, dim), rand(prefix, hk, dim)
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    return dict(q=q.to(DEV), k_cache=k.to(DEV), v_cache=v.to(DEV), lengths=ints(lengths),
                prefix_k=pk.to(DEV), prefix_v=pv.to(DEV), cu_q=ints(cu), slots=ints(slots))


def check(fcv, a, what, scale=None, parts=1, **kw):
    got, lse = fcv.prefix_attention(**a, scale=scale, return_lse=True, **kw)
    q = a["q"]
    cpu = {n: None if t is None else t.cpu() for n, t in a.items() if n != "out"}
    out, want_lse, mass, score, keys = O.prefix_attention(**cpu, scale=scale)
    live = q.shape[0] if a.get("cu_q") is None else int(cpu["cu_q"][-1])
    dim = q.shape[2]
    v_max = max([float(t.nan_to_num(0, 0, 0).abs().max()) for t in
                 (a["v_cache"], a.get("prefix_v")) if t is not None and t.numel()])
    tol = bars.attention(out, mass, score, keys, dim, q.dtype, v_max, parts)
    bars.assert_within(got[:live], out[:live], tol[:live], what)
    bars.assert_within(lse[:live], want_lse[:live], bars.lse(score, keys, dim, want_lse)[:live],
                       what + " lse")
    return got, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,dim", [(14, 2, 64), (4, 4, 64), (8, 2, 128), (40, 1, 64), (3, 1, 128)])
@pytest.mark.parametrize("prefix", [0, 1, 31, 32, 33, 127, 300])
def test_one_token_each(fcv, prefix, hq, hk, dim, dtype):
    lengths = [1, 2, 31, 32, 33, 64, 150, 7]
    say(f"[attn] decode, prefix {prefix}, {hq}/{hk} x {dim} {dtype}")
    a = make([1] * 8, lengths, prefix, hq, hk, dim, dtype)
    got, lse = check(fcv, a, "decode", max_q=1, max_length=150)
    # the same batch without the optional arguments, and with bounds that it passes
    b = dict(a, cu_q=None)
    assert torch.equal(fcv.prefix_attention(**b), check(fcv, b, "no cu_q")[0])
    check(fcv, a, "loose bounds")
    check(fcv, a, "bounds too small", max_q=1, max_length=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,dim", [(14, 2, 64), (8, 8, 64), (8, 2, 128)])
@pytest.mark.parametrize("news,lengths", [
    ([2, 1, 4, 3], [2, 9, 40, 33]),                   # a few tokens each
    ([5, 1, 0, 33, 70], [5, 100, 12, 33, 200]),       # one appends nothing
    ([130, 257, 64], [130, 300, 64]),                 # texts
    ([1, 300], [500, 301]),
])
def test_ragged_appends(fcv, news, lengths, hq, hk, dim, dtype):
    for prefix in (0, 45, 260):
        say(f"[attn] {news} of {lengths} behind {prefix}, {hq}/{hk} x {dim} {dtype}")
        a = make(news, lengths, prefix, hq, hk, dim, dtype)
        check(fcv, a, "append", max_q=max(news), max_length=max(lengths))
        if max(news) > 8:
            check(fcv, a, "max_q too small", max_q=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,dim", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("prefix", [0, 901, 2304])
def test_key_ranges_are_joined(fcv, prefix, hq, hk, dim, dtype):
    """Enough keys for several ranges of the prompt and of the caches; ranges that a short sequence does
    not reach; bounds above and below the lengths."""
    say(f"[attn] ranges, prefix {prefix}, {hq}/{hk} x {dim} {dtype}")
    a = make([1, 2, 1, 3, 1], [1100, 2, 333, 64, 1], prefix, hq, hk, dim, dtype, capacity=1500)
    check(fcv, a, "bounds", max_q=3, max_length=1100)
    check(fcv, a, "capacity", max_q=3)
    check(fcv, a, "too small", max_q=1, max_length=900)
    slot = int(a["slots"][3])
    for value in (float("inf"), -float("inf"), float("nan")):  # the last of three new tokens
        a["v_cache"][slot, 63, 0, 5] = value
        got, _ = check(fcv, a, "hidden", max_q=3, max_length=1100)
        assert got[4:6].isfinite().all() and not got[6, 0, 5].isfinite()


@pytest.mark.parametrize("hq,hk,dim", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("prefix", [0, 512, 2304])
def test_bf16_decode_rounds_the_result_alone(fcv, prefix, hq, hk, dim):
    for sharp in (0.5, 2.0, 8.0):
        say(f"[attn] weights in two parts, prefix {prefix}, {hq}/{hk} x {dim}, sharp {sharp}")
        a = make([1] * 4, [100, 1, 333, 40], prefix, hq, hk, dim, torch.bfloat16, sharp=sharp)
        check(fcv, a, "two parts", parts=2, max_q=1, max_length=333)


def test_many_stacked_rows_behind_a_prompt(fcv):
    """More queries than tiles of 32 take against the prompt, few of each sequence."""
    for dim, hq, hk in ((64, 64, 2), (128, 64, 8)):
        say(f"[attn] 66 x {hq} stacked rows x {dim}")
        lengths = [1 + 13 * i % 70 for i in range(66)]
        a = make([1] * 66, lengths, 900, hq, hk, dim, torch.bfloat16)
        check(fcv, a, "stacked", max_q=1, max_length=max(lengths))


def test_uniform_rows_without_cu_q(fcv):
    for n in (3, 40):
        a = make([n] * 4, [n, 50, 64, 100], 77, 6, 2, 64, torch.float16)
        want = fcv.prefix_attention(**a, max_q=n)
        got, _ = check(fcv, dict(a, cu_q=None), "uniform")
        assert torch.equal(got, want)


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_see_nothing(fcv, dim):
    """No prefix: an empty cache, more queries than keys, a slot outside the caches, a negative
    length."""
    say(f"[attn] empty rows x {dim}")
    news, lengths = [1, 1, 6, 1, 2], [0, 3, 2, 4, -7]
    for prefix in (0, 5):
        a = make(news, [max(n, 0) for n in lengths], prefix, 4, 2, dim, torch.bfloat16)
        a["lengths"] = ints(lengths)
        a["slots"][3] = a["k_cache"].shape[0]
        got, lse = check(fcv, a, f"prefix {prefix}", max_q=6)
        if prefix == 0:
            empty = [0, 2, 3, 4, 5, 8, 9, 10]
            assert (got[empty] == 0).all() and (lse[empty] == -float("inf")).all()
    # nothing at all for anyone
    a = make([1] * 3, [0] * 3, 0, 4, 2, dim, torch.float16)
    got, lse = check(fcv, a, "nothing")
    assert (got == 0).all()
    a.update(prefix_k=None, prefix_v=None)
    assert (fcv.prefix_attention(**a) == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "lowest"])
@pytest.mark.parametrize("n", [3, 40, 200])
def test_hidden_keys_do_not_touch_a_row(fcv, n, bad, dtype):
    """The last new token's key and value are not finite: only the last row may notice.  A value of
    one sign of infinity that a row does see is what it gets."""
    value = torch.finfo(dtype).min if bad == "lowest" else bad
    say(f"[attn] hidden {bad}, {n} new tokens {dtype}")
    for dim in (64, 128):
        a = make([n, 1], [n + 20, 9], 50, 6, 2, dim, dtype)
        slot = int(a["slots"][0])
        a["v_cache"][slot, n + 19, 0, 5] = value
        a["v_cache"][slot, n + 18, 1, 7] = value
        got, _ = check(fcv, {**a, "q": a["q"]}, "values", max_q=n)
        if bad != "lowest":
            assert not got[n - 1, 0, 5].isfinite() and got[:n - 1, 0].isfinite().all()
            assert not got[n - 2:n, 3, 7].isfinite().any() and got[:n - 2, 3].isfinite().all()
        a = make([n, 1], [n + 20, 9], 50, 6, 2, dim, dtype)
        slot = int(a["slots"][0])
        a["k_cache"][slot, n + 19] = value
        got = fcv.prefix_attention(**a, max_q=n)
        clean = make([n, 1], [n + 20, 9], 50, 6, 2, dim, dtype)
        want = fcv.prefix_attention(**clean, max_q=n)
        assert torch.equal(got[:n - 1], want[:n - 1]) and torch.equal(got[n:], want[n:])


def test_large_scores_and_scale(fcv):
    """Scores of hundreds: the running maximum; one row's weights on one key; a scale of its own."""
    for dtype in (torch.bfloat16, torch.float16):
        a = make([1, 9, 1], [300, 77, 1], 400, 4, 2, 64, dtype, sharp=60.0)
        check(fcv, a, "peaked", max_q=9)
        check(fcv, a, "flat", scale=1e-4, max_q=9)
        check(fcv, a, "scale", scale=0.9, max_q=9)


def test_values_near_the_types_largest(fcv):
    """Sums of values near the type's largest stay finite: only their mean has to fit the type."""
    for dtype in (torch.bfloat16, torch.float16):
        a = make([1, 60, 2], [300, 77, 2], 400, 4, 2, 64, dtype)
        for n in ("v_cache", "prefix_v"):
            a[n][:] = a[n].sign() * torch.finfo(dtype).max / 2
        a["v_cache"].nan_to_num_(0)
        a["prefix_v"][:, :, :32] = a["prefix_v"][:, :, :32].abs()
        check(fcv, a, "large", max_q=60)


def test_small_weights_carry_a_long_row(fcv):
    """One key far above thousands of equal ones, whose weights (2^-14 and less of the largest) sum to
    as much as it."""
    for dtype in (torch.float16, torch.bfloat16):
        a = make([1], [4], 6000, 2, 1, 64, dtype)
        a["q"][:] = 0
        a["q"][..., 0] = 8
        a["prefix_k"][:] = 0
        a["prefix_k"][17, 0, 0] = 9.5   # scaled score 9.5: the others' weights are 7.5e-5 of it
        check(fcv, a, "tail")


def test_strides_and_padding(fcv):
    """q inside a packed projection, heads-first caches, keys and values interleaved in one buffer, a
    padded batch."""
    dtype, hq, hk, dim = torch.bfloat16, 6, 2, 64
    say("[attn] strides")
    a = make([1, 3, 2], [40, 33, 100], 70, hq, hk, dim, dtype)
    want = fcv.prefix_attention(**a, max_q=3)
    packed = torch.full((6, (hq + 2 * hk) * dim), float("nan"), dtype=dtype, device=DEV)
    packed[:, :hq * dim] = a["q"].flatten(1)
    b = dict(a, q=packed[:, :hq * dim].unflatten(1, (hq, dim)))
    for n in ("k_cache", "v_cache"):
        b[n] = a[n].transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.stack((a["prefix_k"], a["prefix_v"]), 1)
    b["prefix_k"], b["prefix_v"] = both[:, 0], both[:, 1]
    assert torch.equal(fcv.prefix_attention(**b, max_q=3), want)
    # rows past the last sequence hold NaN and stay; out inside a wider buffer
    q = torch.full((11, hq, dim), float("nan"), dtype=dtype, device=DEV)
    q[:6] = a["q"]
    out = torch.full((11, hq, dim + 8), 7.0, dtype=dtype, device=DEV)
    got, _ = check(fcv, dict(a, q=q), "padded", max_q=3, out=out[..., :dim])
    assert got.data_ptr() == out.data_ptr()
    assert (out[6:] == 7).all() and (out[..., dim:] == 7).all()
    # two sequences that read one session, and one prefix head for all (stride 0)
    c = dict(a, slots=a["slots"].clone())
    c["slots"][2] = c["slots"][1]
    c["lengths"] = ints([40, 33, 33])
    c["prefix_k"] = a["prefix_k"][:, :1].expand(-1, hk, -1)
    check(fcv, c, "shared", max_q=3)
    empty = dict(a, q=a["q"][:0], cu_q=ints([0, 0, 0, 0]))
    assert fcv.prefix_attention(**empty).shape == (0, hq, dim)


def test_a_row_does_not_depend_on_the_batch_beside_it(fcv):
    """Lengths and contents of other sequences do not change a sequence's bits."""
    a = make([1] * 6, [90, 40, 1, 200, 65, 30], 100, 14, 2, 64, torch.bfloat16, capacity=256)
    first = fcv.prefix_attention(**a, max_q=1, max_length=256)
    b = {n: t.clone() for n, t in a.items()}
    b["lengths"][3] = 5
    b["q"][4] = 0
    second = fcv.prefix_attention(**b, max_q=1, max_length=256)
    keep = [0, 1, 2, 5]
    assert torch.equal(first[keep], second[keep])


def test_long_cache_offsets_pass_32_bits(fcv):
    """A cache of 2^31 + elements: the last keys' offsets do not fit 32 bits."""
    cap, hk, dim = (1 << 21) + 64, 8, 128
    say("[attn] caches of 4 GiB")
    k = torch.zeros(1, cap, hk, dim, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(1, hk, dim, generator=g).bfloat16().to(DEV)
    k[0, cap - 9] = q[0] * 4          # nearly all of the weight on one key at the end
    v[0, cap - 9] = torch.randn(hk, dim, generator=g).bfloat16().to(DEV)
    got = fcv.prefix_attention(q, k, v, ints([cap - 8]))
    s = (q[0].double() * k[0, cap - 9].double()).sum(-1) * dim ** -0.5
    w = torch.exp(s) / (torch.exp(s) + cap - 9)
    want = w[:, None] * v[0, cap - 9].double()
    # scores (dim + 4) U * 4 |q|^2 / sqrt(dim) <= 2^-9 here, the weights' rounding, the result's
    assert ((got[0].double() - want).abs() <= 2 ** -6 * want.abs() + 1e-9).all()
    got = fcv.prefix_attention(q, k[:, :8], v[:, :8], ints([0]), prefix_k=k[0, :cap - 8],
                               prefix_v=v[0, :cap - 8])
    assert ((got[0].double() - want).abs() <= 2 ** -6 * want.abs() + 1e-9).all()


def test_bounds_past_32_bits_are_refused(fcv):
    a = make([1, 1], [4, 5], 6, 4, 2, 64, torch.bfloat16)
    for args, match in ((dict(max_q=1 << 31), "range"), (dict(max_length=1 << 31), "range"),
                        (dict(scale=1e300), "scale")):
        with pytest.raises(ValueError, match=match):
            fcv.prefix_attention(**{**a, **args})


def test_refusals(fcv):
    a = make([1, 1], [4, 5], 6, 4, 2, 64, torch.bfloat16)

    def call(**kw):
        return fcv.prefix_attention(**{**a, **kw})

    for args, match in [
            (dict(q=a["q"].float()), "float16 or bfloat16"), (dict(q=a["q"].half()), "k_cache must"),
            (dict(q=a["q"][:, :3]), "multiple of 2"), (dict(q=a["q"][..., :32]), "q must"),
            (dict(v_cache=a["v_cache"][:, :3]), "differ"),
            (dict(k_cache=a["k_cache"][0]), "k_cache must"),
            (dict(lengths=a["lengths"].long()), "lengths must"),
            (dict(lengths=a["lengths"][:0]), "empty"), (dict(cu_q=a["cu_q"][:2]), "cu_q must"),
            (dict(slots=a["slots"][:1]), "slots must"), (dict(prefix_v=None), "together"),
            (dict(prefix_v=a["prefix_v"][:5]), "length"),
            (dict(prefix_k=a["prefix_k"][:, :1]), "prefix_k must"),
            (dict(prefix_k=a["prefix_k"].half(), prefix_v=a["prefix_v"].half()), "prefix_k must"),
            (dict(out=torch.empty(2, 4, 64, device=DEV)), "out must"),
            (dict(out=a["q"][:1].expand(2, 4, 64)), "expanded"), (dict(scale=0.0), "scale"),
            (dict(scale=-1.0), "scale"), (dict(max_q=0), "max_q"),
            (dict(k_cache=a["k_cache"].cpu()), "k_cache must"),
            (dict(q=a["q"].flatten()[4:4 + 256].view(1, 4, 64), cu_q=ints([0, 1, 1])), "16-byte"),
            (dict(q=a["q"][:1], cu_q=None), "divide")]:
        with pytest.raises(ValueError, match=match):
            call(**args)
