"""Operators over many tokens of several sequences against their formulas in 64 bits: rope_tokens, rope_store, attn_packed,
attn_paged (kuiperllama_amd.ops).

Tolerances, from the roundings alone (u = 2^-24, h = half a step of the storage type: 2^-8 for bf16, u for fp32):

  rotation    cosine and sine are off by at most 4 u (angle: two conversions and a product, 3 u of at most 0.79; polynomial: 1.5 u; what
              it leaves out: 0.1 u), their products with the factor, with the elements and the sum of two take 4 u more, and the
              result is rounded once: 8 u f (|a| + |b|) + h |x'|
  attention   a score of n products is off by at most (n + 1) u sum |q k|, its exponent by that times c = scale log2 e and by 3 u
              (|c s| + |c m|) for the fma and its base, the exponential by 2 u more; weights for bf16 are rounded (h); sums of N
              terms take N u.  A weight's relative error e enters the output twice, over the weights and over their sum:
              (2 e + 2 N u + h [bf16]) sum w |v| + 2 h |out|
"""
import math

import pytest
import torch

from test_seq_ops import SCALINGS, frequencies

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rnd(gen, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ---- the formulas ----------------------------------------------------------------------------------------------------
def rotated(x, positions, rot, theta, scaling, half):
    """-> (x', bound of the error of rounding) in 64 bits."""
    f, factor = frequencies(rot, theta, scaling)
    angle = positions.double()[:, None] * torch.tensor(f, dtype=torch.float64, device=x.device)
    cos, sin = (angle.cos() * factor)[:, None, :], (angle.sin() * factor)[:, None, :]
    y, bound = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    i = torch.arange(rot // 2, device=x.device)
    a, b = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
    u, v = x.double()[..., a], x.double()[..., b]
    y[..., a], y[..., b] = u * cos - v * sin, u * sin + v * cos
    # and the table: |position| 2^-54 turns, and this side's own angle, |angle| 2^-53
    bound[..., a] = bound[..., b] = (8 * U + (positions.double().abs() * 2 ** -50)[:, None, None]) * factor * (u.abs() + v.abs())
    return y, bound + half_step(x.dtype) * y.abs() * (1 if rot else 0)


def attended(q, k, v, window, scale):
    """One sequence: n queries at the last n of the keys; -> (out, bound) in 64 bits."""
    n, heads, _ = q.shape
    L, kv = k.shape[:2]
    out = torch.zeros(n, heads, v.shape[2], dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    place = torch.arange(L - n, L, device=q.device)[:, None]
    j = torch.arange(L, device=q.device)[None, :]
    seen = (j <= place) & ((j > place - window) if window > 0 else True)
    any_seen = seen.any(1)
    c = scale * math.log2(math.e)
    h = half_step(q.dtype)
    for head in range(heads):
        kd, vd, qd = k[:, head * kv // heads].double(), v[:, head * kv // heads].double(), q[:, head].double()
        s = (qd @ kd.t()) * scale
        size = (qd.abs() @ kd.abs().t()) * scale
        s = s.masked_fill(~seen, -math.inf)
        m = s.amax(1, keepdim=True).masked_fill(~any_seen[:, None], 0.0)
        p = torch.exp(s - m)
        w = p / p.sum(1, keepdim=True).clamp_min(1e-300)
        out[:, head] = w @ vd
        top = size.masked_fill(~seen, 0.0).amax(1, keepdim=True)  # |s|, |m| are below it too
        e = (q.shape[2] + 1 + 6) * U * top + 4 * U
        bound[:, head] = (2 * e + 2 * L * U + (h if q.dtype == BF16 else 0.0)) * (w @ vd.abs()) + 2 * h * out[:, head].abs()
    return out, bound


def close(got, want, bound, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= bound + 1e-30)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / (bound + 1e-30)).nan_to_num(1e9).max()):.3g} of the bound"


# ---- rotations -------------------------------------------------------------------------------------------------------
ROTATIONS = [  # tokens, heads, kv_heads, size, rot, theta, farthest position
    (1, 32, 8, 64, 64, 5e5, 131072), (33, 14, 2, 64, 64, 1e6, 4096), (5, 6, 6, 48, 48, 1e4, 256), (70, 4, 1, 128, 64, 1e4, 1 << 20),
    (9, 32, 32, 128, 128, 1e4, 4096), (3, 8, 4, 80, 40, 1e4, 8192), (4, 2, 1, 80, 20, 1e4, 8192), (17, 3, 1, 256, 254, 1e4, 4096), (2, 5, 5, 8, 2, 10.0, 99),
    (300, 12, 2, 96, 0, 1e4, 10)]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("half", [True, False], ids=["half", "pairs"])
@pytest.mark.parametrize("shape", ROTATIONS, ids=str)
def test_rotation(gpu, dtype, half, shape):
    from kuiperllama_amd import ops
    T, H, KH, D, rot, theta, far = shape
    gen = generator(T * D + rot)
    rows = rnd(gen, dtype, T, (H + 2 * KH) * D + 16)  # rows that q, k and v are slices of
    q, k, v = (rows[:, a * D:(a + n) * D].view(T, n, D) for a, n in ((0, H), (H, KH), (H + KH, KH)))
    scaling = SCALINGS[(T + D) % len(SCALINGS)]
    pos = torch.randint(0, far, (T,), device=gpu, generator=gen, dtype=torch.int32)
    table = ops.rope_table(rot, theta, gpu, scaling)
    mode = ops.ROPE_HALF if half else ops.ROPE_INTERLEAVED
    wants = [rotated(x, pos, rot, theta, scaling, half) for x in (q, k)]
    before = rows.clone()
    q2, k2 = torch.full((T, H, D), 7.0, dtype=dtype, device=gpu), torch.full((T, KH, D), 7.0, dtype=dtype, device=gpu)
    assert ops.rope_tokens(q, k, pos, table, mode, q_out=q2, k_out=k2)[0] is q2
    assert torch.equal(rows, before)
    close(q2, *wants[0], "q")
    close(k2, *wants[1], "k")
    assert torch.equal(q2[..., rot:], q[..., rot:])
    # into a cache: every place that no token has stays
    page = 16 if T % 2 else 5
    pages = T // page + 3
    kc, vc = (torch.full((pages, KH, page, D), 5.0, dtype=dtype, device=gpu).transpose(1, 2) for _ in range(2))  # heads outside the slots
    slots = torch.randperm(pages * page, device=gpu, generator=gen)[:T].to(torch.int32)
    if T > 2:
        slots[1], slots[2] = -1, pages * page  # nowhere
    kwant, vwant = kc.clone(), vc.clone()
    q3 = torch.full_like(q2, 7.0)
    ops.rope_store(q, k, v, pos, table, mode, kc, vc, slots, q_out=q3)
    for t in range(T):
        s = int(slots[t])
        if 0 <= s < pages * page:
            kwant[s // page, s % page], vwant[s // page, s % page] = k2[t], v[t]
    assert torch.equal(q3, q2) and torch.equal(kc, kwant) and torch.equal(vc, vwant)
    # in place
    ops.rope_tokens(q, k, pos, table, mode)
    assert torch.equal(q, q2) and torch.equal(k, k2)
    assert torch.equal(rows[:, (H + KH) * D:], before[:, (H + KH) * D:])


def test_rotation_far_and_behind(gpu):
    """Positions of either sign up to the ends of int32, where fp32 angles hold nothing."""
    from kuiperllama_amd import ops
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 9, 1 << 24, -(1 << 24) - 1], dtype=torch.int32, device=gpu)
    gen = generator(5)
    q, k = rnd(gen, F32, 8, 3, 64), rnd(gen, F32, 8, 1, 64)
    q2, k2 = torch.empty_like(q), torch.empty_like(k)
    ops.rope_tokens(q, k, pos, ops.rope_table(64, 1e4, gpu), ops.ROPE_HALF, q2, k2)
    close(q2, *rotated(q, pos, 64, 1e4, None, True))
    close(k2, *rotated(k, pos, 64, 1e4, None, True))
    assert torch.equal(q2[0], q[0])  # position 0


# ---- packed prompts --------------------------------------------------------------------------------------------------
def offsets_of(lens, device):
    return torch.tensor([0] + list(torch.tensor(lens, dtype=torch.int64).cumsum(0)), dtype=torch.int32, device=device)


PACKED = [  # heads, kv_heads, key size, value size, lengths, window
    (14, 2, 64, 64, [7, 33, 1], 0), (32, 8, 64, 64, [300, 0, 128, 129, 1, 64], 0), (4, 4, 128, 128, [513], 0), (6, 6, 48, 48, [31, 32, 33, 65], 0),
    (12, 1, 128, 128, [100, 11], 0), (8, 2, 64, 64, [500, 20], 100), (8, 8, 64, 64, [200], 1), (3, 1, 80, 40, [150, 3], 64), (5, 5, 16, 256, [130], 0),
    (4, 2, 256, 256, [140, 70], 37), (7, 1, 192, 128, [90], 0), (2, 1, 8, 8, [40, 1, 1], 0), (1, 1, 64, 64, [1030], 129), (64, 1, 64, 64, [9, 2], 0),
    # few tiles, long prompts: blocks of 32 rows
    (14, 2, 64, 64, [700], 0), (12, 1, 128, 128, [400, 0, 1000], 150), (3, 3, 96, 96, [1000, 385], 0), (2, 1, 256, 192, [500], 0), (5, 1, 40, 72, [901], 300)]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", PACKED, ids=str)
def test_packed(gpu, dtype, case):
    from kuiperllama_amd import ops
    H, KH, D, DV, lens, window = case
    gen = generator(sum(lens) + D)
    T, behind = sum(lens), 3  # rows of a padded batch
    rows = rnd(gen, dtype, T + behind, H * D + KH * (D + DV) + 8)
    q = rows[:, :H * D].view(T + behind, H, D)
    k = rows[:, H * D:(H + KH) * D].view(T + behind, KH, D)
    v = rows[:, (H + KH) * D:(H + KH) * D + KH * DV].view(T + behind, KH, DV)
    out = torch.full((T + behind, H, DV), 9.0, dtype=dtype, device=gpu)
    assert ops.attn_packed(q, k, v, offsets_of(lens, gpu), out, window=window) is out
    first = 0
    for n in lens:
        s = slice(first, first + n)
        if n:
            close(out[s], *attended(q[s], k[s], v[s], window, D ** -0.5), f"length {n}")
        first += n
    assert (out[T:] == 9.0).all()
    if H == KH == 4:  # a scale of one's own
        ops.attn_packed(q, k, v, offsets_of(lens, gpu), out, scale=0.5)
        close(out[:T], *attended(q[:T], k[:T], v[:T], 0, 0.5), "scale")


@pytest.mark.parametrize("n", [150, 900], ids=["tiles", "blocks"])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_what_a_query_does_not_see_does_not_reach_it(gpu, dtype, n):
    """Infinities and NaN in keys and values of later tokens, and of tokens before the window."""
    from kuiperllama_amd import ops
    gen = generator(3)
    H, KH, D, window = 4, 2, 64, 20
    q, k, v = rnd(gen, dtype, n, H, D), rnd(gen, dtype, n, KH, D), rnd(gen, dtype, n, KH, D)
    want, bound = attended(q, k, v, window, D ** -0.5)
    for t, value in ((40, math.inf), (41, math.nan), (75, -math.inf)):
        v[t, :, t % 7::5] = value
    k[100] = math.nan
    k[n - 1, 1, 3] = math.inf
    out = torch.empty(n, H, D, dtype=dtype, device=gpu)
    ops.attn_packed(q, k, v, offsets_of([n], gpu), out, window=window)
    rows = torch.arange(n, device=gpu)
    hit = torch.zeros(n, H, D, dtype=torch.bool, device=gpu)
    for t in (40, 41, 75):
        hit[(rows >= t) & (rows < t + window), :, t % 7::5] = True
    hit[(rows >= 100) & (rows < 100 + window)] = True
    hit[n - 1, 2:] = True
    close(out[~hit], want[~hit], bound[~hit])
    assert not torch.isfinite(out[rows < 100][hit[rows < 100]]).any()
    at40 = out[40, :, 40 % 7::5]
    assert (at40 == math.inf).all()
    assert torch.isnan(out[100:100 + window]).all()


def test_scores_of_any_size(gpu):
    """Rows whose scores differ by thousands, and whose maximum comes late."""
    from kuiperllama_amd import ops
    gen = generator(8)
    n, H, D = 200, 2, 64
    q = rnd(gen, F32, n, H, D)
    k, v = rnd(gen, F32, n, H, D) * torch.linspace(0.1, 60, n, device=gpu)[:, None, None], rnd(gen, F32, n, H, D)
    out = torch.empty_like(q)
    ops.attn_packed(q, k, v, offsets_of([n], gpu), out, scale=1.0)
    close(out, *attended(q, k, v, 0, 1.0))


# ---- a cache of pages ------------------------------------------------------------------------------------------------
def paged(gen, dtype, KH, D, DV, lens, page, spare=3, heads_first=False):
    """A cache whose unused places hold NaN, its table with pages that are none behind each sequence's last, and the keys and values
    of each sequence."""
    held = [-(-n // page) for n in lens]
    total = sum(held) + spare

    def make(size):
        if heads_first:
            return torch.full((total, KH, page, size), math.nan, dtype=dtype, device="cuda").transpose(1, 2)
        return torch.full((total, page, KH, size), math.nan, dtype=dtype, device="cuda")

    kc, vc = make(D), make(DV)
    order = torch.randperm(total, generator=gen, device="cuda")[:sum(held)]
    table = torch.full((len(lens), max(max(held), 1) + 2), -1, dtype=torch.int32, device="cuda")
    at, ks, vs = 0, [], []
    for b, n in enumerate(lens):
        mine = order[at:at + held[b]]
        at += held[b]
        table[b, :held[b]] = mine.to(torch.int32)
        k, v = rnd(gen, dtype, n, KH, D), rnd(gen, dtype, n, KH, DV)
        j = torch.arange(n, device="cuda")
        kc[mine[j // page], j % page], vc[mine[j // page], j % page] = k, v
        ks.append(k)
        vs.append(v)
    return kc, vc, table, ks, vs


PAGED = [  # heads, kv_heads, key size, value size, new tokens, lengths, page, window
    (32, 8, 64, 64, [1] * 5, [1, 16, 17, 700, 64], 16, 0), (32, 8, 128, 128, [1, 1, 1], [4000, 3, 129], 64, 0), (14, 2, 64, 64, [1, 2, 0, 5], [40, 2, 9, 300], 24, 0),
    (8, 2, 64, 64, [200, 1, 33], [900, 1000, 33], 48, 0), (4, 4, 128, 128, [64], [1000], 128, 0), (12, 1, 64, 64, [1, 3], [333, 77], 1, 0),
    (32, 4, 64, 64, [1, 70, 1], [500, 300, 20], 16, 100), (6, 6, 48, 48, [1, 1], [256, 31], 100, 31), (8, 8, 256, 256, [1, 40], [90, 100], 16, 0),
    (3, 1, 80, 40, [2, 9], [50, 9], 7, 5), (2, 2, 64, 64, [3, 1, 4], [1, 0, 4], 16, 0), (64, 1, 128, 128, [1], [600], 32, 0), (1, 1, 16, 16, [1], [5000], 256, 0),
    (32, 8, 64, 64, [8, 4], [515, 1027], 64, 0), (16, 1, 192, 128, [1, 2], [300, 100], 64, 0), (32, 8, 64, 64, [1] * 70, list(range(1, 141, 2)), 16, 0),
    (128, 128, 16, 16, [2200, 1, 40], [2300, 77, 40], 32, 0), (8, 2, 64, 64, [40] * 9 + [1] * 3, [3000, 40, 41, 2000, 777, 90, 64, 1000, 50, 9, 4000, 1], 16, 700),
    (8, 1, 64, 64, [130], [2500], 1, 0)]


def check_paged(q, out, lens, new, ks, vs, window, what=""):
    first, D = 0, q.shape[2]
    for b, (n, length) in enumerate(zip(new, lens)):
        if n > length:  # queries before the first key see nothing
            assert (out[first:first + n - length] == 0).all(), what
            m = length
        else:
            m = n
        if m:
            s = slice(first + n - m, first + n)
            close(out[s], *attended(q[s], ks[b], vs[b], window, D ** -0.5), f"{what} sequence {b}: {n} of {length}")
        first += n


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", PAGED, ids=lambda c: str(c)[:60])
def test_paged(gpu, dtype, case):
    from kuiperllama_amd import ops
    H, KH, D, DV, new, lens, page, window = case
    gen = generator(sum(lens) + D + page)
    kc, vc, table, ks, vs = paged(gen, dtype, KH, D, DV, lens, page, heads_first=len(lens) % 2 == 0)
    T = sum(new)
    q = rnd(gen, dtype, T + 2, H, D, scale=1.5)
    lengths = torch.tensor(lens, dtype=torch.int32, device=gpu)
    ws = ops.attn_paged_workspace(H, KH, DV, T + 2, gpu)
    for max_new in (None, max(new), 1):  # the last may be wrong: it may change no result but by the order of sums
        out = torch.full((T + 2, H, DV), 9.0, dtype=dtype, device=gpu)
        assert ops.attn_paged(q, kc, vc, table, lengths, offsets_of(new, gpu), out, ws, window=window, max_new=max_new) is out
        check_paged(q, out, lens, new, ks, vs, window, f"max_new {max_new}")
        assert (out[T:] == 9.0).all()
    if window:  # pages before the window belong to someone else by now
        for b, (n, length) in enumerate(zip(new, lens)):
            gone = max(0, length - n - window + 1) // page
            table[b, :gone] = torch.tensor([-7, 1 << 30], device=gpu, dtype=torch.int32).repeat(gone)[:gone]
        again = torch.full_like(out, 9.0)
        ops.attn_paged(q, kc, vc, table, lengths, offsets_of(new, gpu), again, ws, window=window, max_new=max_new)
        assert torch.equal(again, out)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 1]], ids=str)
def test_pages_and_lengths_that_are_none(gpu, new):
    """A page number outside the cache and a length behind the table: NaN for the sequence that needs it, the others as ever."""
    from kuiperllama_amd import ops
    gen = generator(21)
    H, KH, D, page, lens = 8, 2, 64, 16, [200, 150, 90]
    kc, vc, table, ks, vs = paged(gen, BF16, KH, D, D, lens, page)
    q = rnd(gen, BF16, sum(new), H, D)
    ws = ops.attn_paged_workspace(H, KH, D, sum(new), gpu)
    off = offsets_of(new, gpu)
    good = torch.empty(sum(new), H, D, dtype=BF16, device=gpu)
    ops.attn_paged(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=gpu), off, good, ws)
    check_paged(q, good, lens, new, ks, vs, 0)
    for number in (-1, kc.shape[0], 2 ** 31 - 1, -2 ** 31):
        broken = table.clone()
        broken[1, 3] = number
        out = torch.zeros_like(good)
        ops.attn_paged(q, kc, vc, broken, torch.tensor(lens, dtype=torch.int32, device=gpu), off, out, ws)
        b = slice(new[0], new[0] + 1)
        assert torch.isnan(out[b]).all() and torch.equal(out[:new[0]], good[:new[0]]) and torch.equal(out[new[0] + 1:], good[new[0] + 1:])
    long = torch.tensor([lens[0], lens[1], table.shape[1] * page + 1000], dtype=torch.int32, device=gpu)
    out = torch.zeros_like(good)
    ops.attn_paged(q, kc, vc, table, long, off, out, ws)
    assert torch.isnan(out[-1]).all() and torch.equal(out[:-1], good[:-1])


def test_sequences_that_share_pages(gpu):
    """Two sequences with the same beginning."""
    from kuiperllama_amd import ops
    gen = generator(4)
    kc, vc, table, ks, vs = paged(gen, F32, 2, 64, 64, [64, 40, 1], 16)
    table[1, :2] = table[0, :2]
    ks[1], vs[1] = torch.cat([ks[0][:32], ks[1][32:]]), torch.cat([vs[0][:32], vs[1][32:]])
    q = rnd(gen, F32, 12, 4, 64)
    out, ws = torch.empty(12, 4, 64, device=gpu), ops.attn_paged_workspace(4, 2, 64, 12, gpu)
    ops.attn_paged(q, kc, vc, table, torch.tensor([64, 40, 1], dtype=torch.int32, device=gpu), offsets_of([1, 10, 1], gpu), out, ws)
    check_paged(q, out, [64, 40, 1], [1, 10, 1], ks, vs, 0)


# ---- together --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_a_layer_s_attention_in_portions(gpu, dtype):
    """Three prompts, whole, against the same tokens in portions over a cache, then single tokens in a captured graph whose lengths,
    slots and positions move on the device."""
    from kuiperllama_amd import ops
    gen = generator(77)
    H, KH, D, page, lens, steps = 8, 2, 64, 16, [150, 37, 90], 6
    whole = [n + steps for n in lens]
    raw = [(rnd(gen, dtype, n, H, D, scale=2.0), rnd(gen, dtype, n, KH, D), rnd(gen, dtype, n, KH, D)) for n in whole]
    table = ops.rope_table(D, 5e5, gpu, SCALINGS[3])
    mode = ops.ROPE_HALF
    # whole prompts
    q, k, v = (torch.cat([r[i] for r in raw]) for i in range(3))
    pos = torch.cat([torch.arange(n, device=gpu, dtype=torch.int32) for n in whole])
    qr, kr = torch.empty_like(q), torch.empty_like(k)
    ops.rope_tokens(q, k, pos, table, mode, qr, kr)
    want = torch.empty_like(q)
    ops.attn_packed(qr, kr, v, offsets_of(whole, gpu), want)
    first = [0, whole[0], whole[0] + whole[1]]
    bounds = [attended(qr[f:f + n], kr[f:f + n], v[f:f + n], 0, D ** -0.5) for f, n in zip(first, whole)]
    for b in range(3):
        close(want[first[b]:first[b] + whole[b]], *bounds[b], "whole")
    # portions
    held = [-(-n // page) for n in whole]
    kc = torch.full((sum(held) + 1, page, KH, D), math.nan, dtype=dtype, device=gpu)
    vc = torch.full_like(kc, math.nan)
    pages = torch.zeros(3, max(held), dtype=torch.int32, device=gpu)
    order = torch.randperm(sum(held), device=gpu, generator=gen).to(torch.int32)
    for b, part in enumerate(order.split(held)):
        pages[b, :held[b]] = part
    done = [0, 0, 0]
    for portion in ([64, 37, 1], [60, 0, 89], [26, 0, 0]):
        x = [torch.cat([raw[b][i][done[b]:done[b] + portion[b]] for b in range(3)]) for i in range(3)]
        p = torch.cat([torch.arange(done[b], done[b] + portion[b], device=gpu, dtype=torch.int32) for b in range(3)])
        seq = torch.cat([torch.full((portion[b],), b, device=gpu) for b in range(3)])
        slots = pages[seq, p.long() // page] * page + p % page
        ops.rope_store(x[0], x[1], x[2], p, table, mode, kc, vc, slots)
        done = [a + n for a, n in zip(done, portion)]
        out, ws = torch.empty_like(x[0]), ops.attn_paged_workspace(H, KH, D, sum(portion), gpu)
        ops.attn_paged(x[0], kc, vc, pages, torch.tensor(done, dtype=torch.int32, device=gpu), offsets_of(portion, gpu), out, ws)
        at = 0
        for b in range(3):
            s = slice(done[b] - portion[b], done[b])
            close(out[at:at + portion[b]], bounds[b][0][s], bounds[b][1][s], f"portion of {b}")
            at += portion[b]
    # single tokens, captured
    sq, sk, sv = (torch.zeros(3, n, D, dtype=dtype, device=gpu) for n in (H, KH, KH))
    spos, slen, sslots = (torch.zeros(3, dtype=torch.int32, device=gpu) for _ in range(3))
    soff, sout, ws = offsets_of([1, 1, 1], gpu), torch.zeros(3, H, D, dtype=dtype, device=gpu), ops.attn_paged_workspace(H, KH, D, 3, gpu)

    def step():
        ops.rope_store(sq, sk, sv, spos, table, mode, kc, vc, sslots)
        ops.attn_paged(sq, kc, vc, pages, slen, soff, sout, ws, max_new=1)

    graph = None
    for i in range(steps):
        for b in range(3):
            sq[b], sk[b], sv[b] = raw[b][0][done[b]], raw[b][1][done[b]], raw[b][2][done[b]]
        spos.copy_(torch.tensor(done, dtype=torch.int32))
        slen.copy_(spos + 1)
        sslots.copy_(pages[torch.arange(3, device=gpu), spos.long() // page] * page + spos % page)
        if i == 0:
            keep = [t.clone() for t in (sq, sk)]
            step()
            torch.cuda.synchronize()
            eager = sout.clone()
            sq.copy_(keep[0])
            sout.zero_()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
            graph.replay()
            assert torch.equal(sout, eager)
        else:
            sout.fill_(math.nan)
            torch.cuda.synchronize()
            graph.replay()
        for b in range(3):
            close(sout[b:b + 1], bounds[b][0][done[b]:done[b] + 1], bounds[b][1][done[b]:done[b] + 1], f"step {i} of {b}")
        done = [n + 1 for n in done]


# ---- units and tiles that are cut: long keys, few sequences ------------------------------------------------------------------
CUT = [  # heads, kv_heads, key size, value size, new tokens, lengths, page: single tokens dealt by steps of keys, portions cut into parts
    (8, 1, 64, 64, [1], [20000], 16), (4, 1, 128, 128, [2, 1], [9000, 5], 16), (2, 1, 256, 256, [1], [3000], 32), (4, 2, 48, 80, [1, 3], [2500, 1], 8),
    (8, 1, 64, 64, [200], [6000], 3), (4, 2, 128, 128, [300, 1], [4000, 2000], 16), (4, 1, 256, 256, [60, 40, 1], [1500, 2100, 700], 32),
    (8, 2, 128, 96, [257], [1700], 24),
    (8, 8, 64, 64, [33] * 70 + [1] * 3, [90] * 70 + [1, 200, 3000], 16), (6, 6, 16, 256, [40] * 101, [57] * 101, 8)]  # more tiles than workgroups


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", CUT, ids=lambda c: str(c)[:60])
def test_cut_keys(gpu, dtype, case):
    """Against the formula; a page that is none in one of the parts; values that are no numbers in keys that some rows do not see."""
    from kuiperllama_amd import ops
    H, KH, D, DV, new, lens, page = case
    gen = generator(sum(lens) + D)
    kc, vc, table, ks, vs = paged(gen, dtype, KH, D, DV, lens, page)
    T = sum(new)
    q = rnd(gen, dtype, T, H, D, scale=1.5)
    lengths, off = torch.tensor(lens, dtype=torch.int32, device=gpu), offsets_of(new, gpu)
    ws = ops.attn_paged_workspace(H, KH, DV, T, gpu)

    def run(pages):
        out = torch.full((T, H, DV), 9.0, dtype=dtype, device=gpu)
        return ops.attn_paged(q, kc, vc, pages, lengths, off, out, ws)

    good = run(table)
    check_paged(q, good, lens, new, ks, vs, 0)
    assert torch.equal(run(table), good)
    for at in (1, lens[0] // page // 2):  # of the first sequence
        broken = table.clone()
        broken[0, at] = -5
        out = run(broken)
        assert torch.isnan(out[:new[0]]).all() and torch.equal(out[new[0]:], good[new[0]:])
    assert torch.equal(run(table), good)
    # the last token of the first sequence, and one in the middle of its new ones, hold what is no number
    n, length = new[0], lens[0]
    spoilt = torch.zeros(T, H, DV, dtype=torch.bool, device=gpu)
    for place, value in ((length - 1, math.nan), (length - 1 - n // 2, -math.inf)):
        pg = int(table[0, place // page])
        vc[pg, place % page, 0, ::3] = value
        spoilt[max(0, place - (length - n)):n, :H // KH, ::3] = True
    out = run(table)
    assert not torch.isfinite(out[spoilt]).any()
    want, bound = attended(q[:n], ks[0], vs[0], 0, D ** -0.5)
    close(out[:n][~spoilt[:n]], want[~spoilt[:n]], bound[~spoilt[:n]], "beside what is no number")
    assert torch.equal(out[n:], good[n:])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 2, 1], [70, 1, 40]], ids=str)
def test_one_cache_tensor_and_a_window(gpu, dtype, new):
    """Keys and values side by side in one tensor, queries a slice of wider rows, every length of the last page."""
    from kuiperllama_amd import ops
    gen = generator(31 + sum(new))
    H, KH, D, page, window = 6, 2, 64, 16, 50
    T = sum(new)
    for extra in range(0, page, 5):
        lens = [300 + extra, max(new[1], 33) + extra, 41 + extra]
        kc, vc, table, ks, vs = paged(gen, dtype, KH, D, D, lens, page)
        both = torch.stack([kc, vc], 2)  # [pages, page, 2, kv_heads, size]
        rows = rnd(gen, dtype, T, 2, H, D)
        out = torch.full((T, 2, H, D), 9.0, dtype=dtype, device=gpu)
        ops.attn_paged(rows[:, 1], both[:, :, 0], both[:, :, 1], table, torch.tensor(lens, dtype=torch.int32, device=gpu), offsets_of(new, gpu), out[:, 0],
                       ops.attn_paged_workspace(H, KH, D, T, gpu), window=window)
        check_paged(rows[:, 1], out[:, 0], lens, new, ks, vs, window, f"extra {extra}")
        assert (out[:, 1] == 9.0).all()


def test_keys_that_heads_share_by_a_stride_of_zero(gpu):
    from kuiperllama_amd import ops
    gen = generator(6)
    q, k, v = rnd(gen, BF16, 90, 4, 64), rnd(gen, BF16, 90, 1, 64), rnd(gen, BF16, 90, 1, 64)
    a, b = (ops.attn_packed(q, x, y, offsets_of([70, 20], gpu), torch.empty_like(q)) for x, y in ((k, v), (k.expand(-1, 4, -1), v.expand(-1, 4, -1))))
    close(a[:70], *attended(q[:70], k[:70], v[:70], 0, 0.125))
    close(b[:70], *attended(q[:70], k[:70], v[:70], 0, 0.125))
    close(b[70:], *attended(q[70:], k[70:], v[70:], 0, 0.125))


def test_no_tokens(gpu):
    from kuiperllama_amd import ops
    f = lambda *s: torch.zeros(*s, dtype=BF16, device=gpu)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)  # noqa: E731
    table = ops.rope_table(64, 1e4, gpu)
    ops.rope_tokens(f(0, 4, 64), f(0, 2, 64), i(0), table, 1)
    ops.rope_store(f(0, 4, 64), f(0, 2, 64), f(0, 2, 64), i(0), table, 1, f(3, 16, 2, 64), f(3, 16, 2, 64), i(0))
    ops.attn_packed(f(0, 4, 64), f(0, 2, 64), f(0, 2, 64), i(1), f(0, 4, 64))
    ws = ops.attn_paged_workspace(4, 2, 64, 0, gpu)
    ops.attn_paged(f(0, 4, 64), f(3, 16, 2, 64), f(3, 16, 2, 64), i(2, 3), i(2), i(3), f(0, 4, 64), ws)
    out = f(5, 4, 64) + 9  # a padded batch of no sequence
    ops.attn_packed(f(5, 4, 64), f(5, 2, 64), f(5, 2, 64), i(1), out)
    ops.attn_paged(f(5, 4, 64), f(3, 16, 2, 64), f(3, 16, 2, 64), i(0, 3), i(0), i(1), out, ops.attn_paged_workspace(4, 2, 64, 5, gpu))
    assert (out == 9).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_one_workspace_for_calls_of_any_shape(gpu, dtype):
    """Two captured graphs and eager calls of other shapes, one after the other, over one workspace; lengths move between replays."""
    from kuiperllama_amd import ops
    gen = generator(55)
    KH, D, page = 2, 64, 16
    lens = [[2000, 5, 900], [1500, 2500]]
    news = [[1, 1, 1], [90, 40]]
    caches = [paged(gen, dtype, KH, D, D, n, page) for n in lens]
    qs = [rnd(gen, dtype, sum(n), 8, D) for n in news]
    ws = ops.attn_paged_workspace(8, KH, D, 130, gpu)
    lengths = [torch.tensor(n, dtype=torch.int32, device=gpu) for n in lens]
    offs = [offsets_of(n, gpu) for n in news]
    outs = [torch.zeros_like(q) for q in qs]

    def call(i, out):
        kc, vc, table = caches[i][:3]
        ops.attn_paged(qs[i], kc, vc, table, lengths[i], offs[i], out, ws, max_new=max(news[i]))

    for i in range(2):
        call(i, outs[i])
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(i, outs[i])
        graphs.append(g)
    for turn in range(6):
        now = [[n - 13 * turn if n > 100 else n for n in x] for x in lens]
        for i in range(2):
            lengths[i].copy_(torch.tensor(now[i], dtype=torch.int32))
            outs[i].fill_(math.nan)
        order = (0, 1) if turn % 2 else (1, 0)
        for i in order:
            graphs[i].replay()
        eager = [torch.zeros_like(o) for o in outs]
        for i in order:
            call(i, eager[i])
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], eager[i]), turn
            ks, vs = ([x[:n] for x, n in zip(t, now[i])] for t in caches[i][3:])
            check_paged(qs[i], outs[i], now[i], news[i], ks, vs, 0, f"turn {turn}")
    assert not ws[:4096].any()  # the counters, as the next call needs them


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("max_new", [None, 1], ids=["tiles", "rows"])
def test_more_new_tokens_than_keys_and_rows_ahead_of_the_first_sequence(gpu, dtype, max_new):
    """Queries ahead of a sequence's first key get zeros, in tiles and in parts of them; rows that belong to no sequence stay."""
    from kuiperllama_amd import ops
    gen = generator(66)
    H, KH, D, page, ahead = 4, 2, 64, 16, 7
    new, lens = [200, 150, 90, 1], [70, 0, 2000, 1]
    kc, vc, table, ks, vs = paged(gen, dtype, KH, D, D, lens, page)
    q = rnd(gen, dtype, ahead + sum(new) + 4, H, D)
    out = torch.full_like(q, 9.0)
    ops.attn_paged(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=gpu), offsets_of(new, gpu) + ahead, out,
                   ops.attn_paged_workspace(H, KH, D, q.shape[0], gpu), max_new=max_new)
    check_paged(q[ahead:], out[ahead:], lens, new, ks, vs, 0)
    assert (out[:ahead] == 9.0).all() and (out[ahead + sum(new):] == 9.0).all()
    k, v = rnd(gen, dtype, q.shape[0], KH, D), rnd(gen, dtype, q.shape[0], KH, D)
    out.fill_(9.0)
    ops.attn_packed(q, k, v, offsets_of(new, gpu) + ahead, out)
    for b, n in enumerate(new):
        s = slice(ahead + sum(new[:b]), ahead + sum(new[:b + 1]))
        close(out[s], *attended(q[s], k[s], v[s], 0, D ** -0.5), f"packed {n}")
    assert (out[:ahead] == 9.0).all() and (out[ahead + sum(new):] == 9.0).all()


@pytest.mark.parametrize("power", [-100, 100])
def test_fp32_of_any_size(gpu, power):
    """Values near both ends of the exponents: as exact as those near one."""
    from kuiperllama_amd import ops
    gen = generator(14)
    n, H, D = 130, 2, 64
    q, k, v = rnd(gen, F32, n, H, D), rnd(gen, F32, n, H, D), rnd(gen, F32, n, H, D)
    want, bound = attended(q, k, v, 0, D ** -0.5)
    out = ops.attn_packed(q * 2.0 ** -60, k * 2.0 ** 60, v * 2.0 ** power, offsets_of([n], gpu), torch.empty_like(q))
    close(out.double() * 2.0 ** -power, want, bound)


def test_another_stream_and_the_same_answer_twice(gpu):
    from kuiperllama_amd import ops
    gen = generator(12)
    kc, vc, table, ks, vs = paged(gen, BF16, 2, 128, 128, [3000, 5, 800], 64)
    q = rnd(gen, BF16, 3, 8, 128)
    lengths, off = torch.tensor([3000, 5, 800], dtype=torch.int32, device=gpu), offsets_of([1, 1, 1], gpu)
    ws = [ops.attn_paged_workspace(8, 2, 128, 3, gpu) for _ in range(2)]
    outs = [torch.zeros(3, 8, 128, dtype=BF16, device=gpu) for _ in range(2)]
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(side[i]):
                ops.attn_paged(q, kc, vc, table, lengths, off, outs[i], ws[i])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])
    check_paged(q, outs[0], [3000, 5, 800], [1, 1, 1], ks, vs, 0)


def test_offsets_past_32_bits(gpu):
    """A cache of more than 4 GiB: pages at its end."""
    from kuiperllama_amd import ops
    pages, page, KH, D = 70000, 256, 1, 128
    kc = torch.zeros(pages, page, KH, D, dtype=BF16, device=gpu)  # 4.6 GB
    vc = torch.zeros(pages, page, KH, D, dtype=BF16, device=gpu)
    gen = generator(9)
    ids = [69999, 3, 65536, 69998]
    n = 1000
    k, v = rnd(gen, BF16, n, KH, D), rnd(gen, BF16, n, KH, D)
    slots = torch.tensor([ids[j // page] * page + j % page for j in range(n)], dtype=torch.int32, device=gpu)
    q = rnd(gen, BF16, n, 4, D)
    table = ops.rope_table(0, 1e4, gpu)  # nothing turns
    ops.rope_store(q, k, v, torch.zeros(n, dtype=torch.int32, device=gpu), table, 0, kc, vc, slots)
    assert torch.equal(kc[69998, :n - 768], k[768:]) and torch.equal(vc[69999], v[:256])
    ws = ops.attn_paged_workspace(4, KH, D, n, gpu)
    out = torch.empty(n, 4, D, dtype=BF16, device=gpu)
    args = (kc, vc, torch.tensor([ids], dtype=torch.int32, device=gpu), torch.tensor([n], dtype=torch.int32, device=gpu))
    ops.attn_paged(q, *args, offsets_of([n], gpu), out, ws)
    want, bound = attended(q, k, v, 0, D ** -0.5)
    close(out, want, bound)
    ops.attn_paged(q[-1:], *args, offsets_of([1], gpu), out[-1:], ws)
    close(out[-1:], want[-1:], bound[-1:])


def test_refusals_on_the_device(gpu):
    from kuiperllama_amd import _ffi, ops
    f = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device=gpu)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)  # noqa: E731
    table = ops.rope_table(64, 1e4, gpu)
    ok = dict(q=f(4, 4, 64), k=f(4, 2, 64), positions=i(4), table=table, mode=1)
    for bad, error in ((dict(q=f(4, 4, 64, dtype=torch.float16)), TypeError), (dict(k=f(4, 2, 64, dtype=F32)), TypeError), (dict(k=f(3, 2, 64)), ValueError),
                       (dict(k=f(4, 2, 128)), ValueError), (dict(positions=i(3)), ValueError), (dict(positions=f(4, dtype=F32)), TypeError),
                       (dict(q_out=f(4, 4, 32)), ValueError), (dict(q=f(4, 64, 4).transpose(1, 2)), ValueError), (dict(mode=5), _ffi.KhError),
                       (dict(q=f(4, 4, 65)[..., 1:]), _ffi.KhError), (dict(k=f(4, 3, 64)), _ffi.KhError), (dict(positions=torch.zeros(4, dtype=torch.int32)), ValueError),
                       (dict(q=f(4, 256)), ValueError)):
        with pytest.raises(error):
            ops.rope_tokens(**{**ok, **bad})
    ok = dict(q=f(4, 4, 64), kcache=f(3, 16, 2, 64), vcache=f(3, 16, 2, 64), pages=i(2, 3), lengths=i(2), offsets=i(3), out=f(4, 4, 64),
              workspace=ops.attn_paged_workspace(4, 2, 64, 4, gpu))
    for bad, error in ((dict(lengths=i(3)), ValueError), (dict(pages=i(3, 3)), ValueError), (dict(pages=i(2, 3).long()), TypeError), (dict(out=f(4, 4, 32)), ValueError),
                       (dict(vcache=f(3, 8, 2, 64)), ValueError), (dict(kcache=f(3, 16, 2, 32)), ValueError), (dict(workspace=f(0).to(torch.uint8)), _ffi.KhError),
                       (dict(scale=0.0), _ffi.KhError), (dict(kcache=f(3, 16, 2, 64, dtype=F32)), TypeError), (dict(offsets=i(3).long()), TypeError),
                       (dict(workspace=torch.zeros(1 << 20, dtype=torch.uint8)), ValueError), (dict(max_new=-1), _ffi.KhError)):
        with pytest.raises(error):
            ops.attn_paged(**{**ok, **bad})
    assert (ops.attn_paged(**ok) == 0).all()  # offsets and lengths of zero
    ok = dict(q=f(4, 4, 64), k=f(4, 2, 64), v=f(4, 2, 64), offsets=i(2), out=f(4, 4, 64))
    for bad, error in ((dict(k=f(3, 2, 64)), ValueError), (dict(v=f(4, 1, 64)), ValueError), (dict(v=f(4, 2, 64, dtype=F32)), TypeError), (dict(out=f(4, 4, 64, dtype=F32)), TypeError),
                       (dict(k=f(4, 3, 64), v=f(4, 3, 64)), _ffi.KhError), (dict(q=f(4, 4, 320), k=f(4, 2, 320)), _ffi.KhError)):
        with pytest.raises(error):
            ops.attn_packed(**{**ok, **bad})


# ---- every way that a call can be dealt ------------------------------------------------------------------------------------
def every_form(q, k, v, **kw):
    """One sequence, as a whole prompt (150 tokens: tiles, 900: blocks of 32 rows), as the last two thirds of it over pages in tiles and in
    rows, its last token alone.  -> name, first token, out"""
    from kuiperllama_amd import ops
    n, H = q.shape[:2]
    KH, DV = v.shape[1:]
    yield "packed", 0, ops.attn_packed(q, k, v, offsets_of([n], q.device), torch.full((n, H, DV), 9.0, dtype=q.dtype, device=q.device), **kw)
    page, j = 16, torch.arange(n, device=q.device)
    held = -(-n // page)
    at = held - 1 - j // page, j % page  # the pages from behind
    kc, vc = (torch.full((held, page, KH, x.shape[2]), math.nan, dtype=q.dtype, device=q.device) for x in (k, v))
    kc[at], vc[at] = k, v
    table = torch.arange(held - 1, -1, -1, dtype=torch.int32, device=q.device)[None]
    length = torch.tensor([n], dtype=torch.int32, device=q.device)
    for name, new, most in (("portion", n - n // 3, None), ("rows", n - n // 3, 1), ("last", 1, 1)):
        out = torch.full((new, H, DV), 9.0, dtype=q.dtype, device=q.device)
        ws = ops.attn_paged_workspace(H, KH, DV, new, q.device)
        yield name, n - new, ops.attn_paged(q[n - new:], kc, vc, table, length, offsets_of([new], q.device), out, ws, max_new=most, **kw)


@pytest.mark.parametrize("n", [150, 900], ids=["tiles", "blocks"])
def test_weights_add_up_to_one(gpu, n):
    """Values that are the same in every token come out as they are, whatever bf16 makes of the weights: their sum is taken of the rounded ones.
    One key outweighs the others by 2^2 to 2^3 and comes after a tile of theirs, so that its own weight is no power of two and is rounded.
    The sums of n terms are off by 2 n u of the value at most (900: 1.1e-4), and a value's nearest other rounding is 2^-9 of it away."""
    gen = generator(91)
    H, KH, D = 16, 16, 64
    q, k = torch.zeros(n, H, D, dtype=BF16, device=gpu), torch.zeros(n, KH, D, dtype=BF16, device=gpu)
    q[..., 0] = 1
    k[..., 0] = -20
    k[0, :, 0] = 0
    k[130, :, 0] = 2 + (2 * torch.arange(KH, device=gpu) + 1) / 64
    v = rnd(gen, BF16, 1, KH, D).expand(n, -1, -1).contiguous()
    for name, first, out in every_form(q, k, v, scale=math.log(2.0)):
        assert torch.equal(out, v[first:]), name


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("max_new", [None, 1], ids=["tiles", "rows"])
def test_a_window_that_holds_everything(gpu, dtype, max_new):
    """The largest int32 as a window, with queries ahead of their sequence's first key too: as no window."""
    from kuiperllama_amd import ops
    gen = generator(67)
    H, KH, D, page = 4, 2, 64, 16
    new, lens = [200, 150, 90, 1], [70, 0, 2000, 30]
    kc, vc, table, ks, vs = paged(gen, dtype, KH, D, D, lens, page)
    q = rnd(gen, dtype, sum(new), H, D)
    ws = ops.attn_paged_workspace(H, KH, D, q.shape[0], gpu)
    args = (q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=gpu), offsets_of(new, gpu))
    want = ops.attn_paged(*args, torch.full_like(q, 9.0), ws, max_new=max_new)
    check_paged(q, want, lens, new, ks, vs, 0)
    for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30, 2 ** 30 - 1, 5000):
        out = ops.attn_paged(*args, torch.full_like(q, 9.0), ws, max_new=max_new, window=window)
        check_paged(q, out, lens, new, ks, vs, 0, f"window {window}")
        assert torch.equal(out, want), window


BOTH = [pytest.mark.parametrize("n", [150, 900], ids=["tiles", "blocks"]), pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])]


def both(f):
    for mark in BOTH:
        f = mark(f)
    return f


@both
def test_scores_that_are_all_minus_infinity(gpu, dtype, n):
    """A query that sees keys, every one of them at minus infinity, has no softmax: NaN, as the formula says, and not the zeros of a query that
    sees none.  One finite key is enough."""
    gen = generator(92)
    H, KH, D, t = 4, 2, 64, 100
    q, k, v = rnd(gen, dtype, n, H, D), rnd(gen, dtype, n, KH, D), rnd(gen, dtype, n, KH, D)
    q[..., 0] = q[..., 0].abs() + 1
    k[:t, :, 0] = -math.inf
    want, bound = attended(q[t:], k[t:], v[t:], 0, D ** -0.5)
    for name, first, out in every_form(q, k, v):
        none = max(0, t - first)
        assert torch.isnan(out[:none]).all(), name
        close(out[none:], want[first + none - t:], bound[first + none - t:], name)
    k[:, :, 0] = -math.inf
    for name, first, out in every_form(q, k, v):
        assert torch.isnan(out).all(), name


@both
def test_an_infinity_of_a_weight_that_vanishes(gpu, dtype, n):
    """A key that a query sees, of a weight that fp32 has no number for: its infinity is not lost."""
    gen = generator(94)
    H, KH, D, t = 4, 2, 64, 5
    q, k, v = torch.zeros(n, H, D, dtype=dtype, device=gpu), torch.zeros(n, KH, D, dtype=dtype, device=gpu), rnd(gen, dtype, n, KH, D)
    q[..., 0] = 1
    k[t, :, 0] = -300
    want, bound = attended(q, k, v, 0, 1.0)
    v[t, :, ::3] = math.inf
    hit = torch.zeros(n, H, D, dtype=torch.bool, device=gpu)
    hit[t:, :, ::3] = True
    for name, first, out in every_form(q, k, v, scale=1.0):
        assert not torch.isfinite(out[hit[first:]]).any(), name
        close(out[~hit[first:]], want[first:][~hit[first:]], bound[first:][~hit[first:]], name)


@both
def test_means_of_values_near_the_largest_number(gpu, dtype, n):
    """Values of 2^127 to 1.9 2^127: their sum has no room in fp32, their mean has."""
    gen = generator(93)
    H, KH, D = 4, 2, 64
    q, k = rnd(gen, dtype, n, H, D), rnd(gen, dtype, n, KH, D)
    v = (1 + 0.9 * torch.rand(n, KH, D, device=gpu, generator=gen)) * 2.0 ** 127
    v[..., 1::2] *= (torch.rand(n, KH, D // 2, device=gpu, generator=gen) < 0.5) * 2.0 - 1
    v = v.to(dtype)
    want, bound = attended(q, k, v, 0, D ** -0.5)
    for name, first, out in every_form(q, k, v):
        assert torch.isfinite(out).all(), name
        close(out, want[first:], bound[first:], name)


@both
def test_scores_near_the_largest_number(gpu, dtype, n):
    """Scores of 3e38 that are all alike have equal weights; smaller ones beside them have none."""
    gen = generator(95)
    H, KH, D = 4, 2, 64
    q, k, v = torch.zeros(n, H, D, dtype=dtype, device=gpu), torch.zeros(n, KH, D, dtype=dtype, device=gpu), rnd(gen, dtype, n, KH, D)
    q[..., 0] = 2.0 ** 64
    k[..., 0] = 1.75 * 2.0 ** 63
    k[1::3, :, 0] = -(2.0 ** 63)
    want, bound = attended(torch.ones_like(q[..., :1]), (k[..., :1] > 0).to(dtype) * 1000, v, 0, 1.0)
    for name, first, out in every_form(q, k, v, scale=1.0):
        close(out, want[first:], bound[first:], name)


@both
def test_a_query_that_is_no_number_leaves_the_others_as_they_are(gpu, dtype, n):
    """Bit for bit: rows that share a product with it are not done in another order for it."""
    gen = generator(96)
    H, KH, D = 8, 2, 64
    q, k, v = rnd(gen, dtype, n, H, D), rnd(gen, dtype, n, KH, D), rnd(gen, dtype, n, KH, D)
    broken = q.clone()
    broken[77, 1], broken[n - 1, 5, 3] = math.nan, math.nan
    for (name, first, good), (_, _, out) in zip(every_form(q, k, v), every_form(broken, k, v)):
        hit = torch.isnan(broken[first:]).any(-1)
        assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], good[~hit]), name


def test_outputs_of_any_layout_without_overlaps(gpu):
    """Heads outside tokens, wider rows, one token with any stride, pages within slots: as contiguous ones; expanded tensors are refused."""
    from kuiperllama_amd import _ffi, ops
    gen = generator(97)
    T, H, KH, D, pages, page = 20, 4, 2, 64, 5, 16
    q, k, v = rnd(gen, BF16, T, H, D), rnd(gen, BF16, T, KH, D), rnd(gen, BF16, T, KH, D)
    off, pos = offsets_of([T], gpu), torch.arange(T, dtype=torch.int32, device=gpu)
    table = ops.rope_table(D, 1e4, gpu)
    empty = lambda *s: torch.zeros(*s, dtype=BF16, device=gpu)  # noqa: E731
    want = ops.attn_packed(q, k, v, off, empty(T, H, D))
    for out in (empty(H, T, D).transpose(0, 1), empty(T, H, 2 * D)[..., D:], empty(T, 3, H, D)[:, 1]):
        assert torch.equal(ops.attn_packed(q, k, v, off, out), want)
    one = ops.attn_packed(q[:1], k[:1], v[:1], offsets_of([1], gpu), empty(1, H, D).as_strided((1, H, D), (0, D, 1)))
    assert torch.equal(one, want[:1])
    wants = ops.rope_tokens(q, k, pos, table, ops.ROPE_HALF, empty(T, H, D), empty(T, KH, D))
    got = ops.rope_tokens(q, k, pos, table, ops.ROPE_HALF, empty(H, T, D).transpose(0, 1), empty(KH, T, D).transpose(0, 1))
    assert torch.equal(got[0], wants[0]) and torch.equal(got[1], wants[1])
    caches = []
    for make in (lambda: empty(pages, page, KH, D), lambda: empty(page, KH, pages, D).permute(2, 0, 1, 3), lambda: empty(KH, pages, page, D).permute(1, 2, 0, 3)):
        kc, vc = make(), make()
        ops.rope_store(q, k, v, pos, table, ops.ROPE_HALF, kc, vc, pos, q_out=empty(T, H, D))
        caches.append((kc, vc))
    for kc, vc in caches[1:]:
        assert torch.equal(kc, caches[0][0]) and torch.equal(vc, caches[0][1])
    for bad in (lambda: ops.attn_packed(q, k, v, off, empty(T, 1, D).expand(T, H, D)), lambda: ops.attn_packed(q, k, v, off, empty(1, H, D).expand(T, H, D)),
                lambda: ops.rope_tokens(q, k[:, :1].expand(T, KH, D), pos, table, ops.ROPE_HALF), lambda: ops.attn_packed(q, q, q, off, q),
                lambda: ops.rope_store(q, k, v, pos, table, ops.ROPE_HALF, empty(pages, page, 1, D).expand(pages, page, KH, D), empty(pages, page, KH, D), pos)):
        with pytest.raises(_ffi.KhError):
            bad()


# ---- tiles enough for the chip, sequences by the hundred -------------------------------------------------------------------
MANY = [  # heads, kv_heads, key size, value size, new tokens, lengths, page, window
    (32, 8, 128, 128, [2100], [2900], 16, 0), (32, 8, 128, 128, [1500, 650], [1500, 900], 24, 333),  # 525 tiles
    (64, 64, 96, 96, [1100, 1], [1300, 500], 16, 0), (64, 64, 80, 80, [1100], [1200], 7, 100),  # 550
    (64, 64, 256, 256, [600], [800], 16, 0), (40, 40, 192, 128, [840, 3], [900, 77], 1, 0),  # 300 and 280, of 256 columns
    (8, 2, 96, 96, [100, 1, 40], [1000, 300, 40], 16, 0), (8, 2, 80, 88, [150], [700], 5, 90),  # a portion of 65 to 96 columns, in parts
    (4, 2, 64, 64, [1] * 600, [1 + 37 * b % 419 for b in range(600)], 16, 0), (4, 1, 128, 128, [b % 3 for b in range(300)], [b % 3 + b for b in range(300)], 16, 50),
    (2, 1, 64, 64, [1] * 500 + [60] + [1] * 550 + [40], [1 + b % 61 for b in range(500)] + [600] + [3] * 550 + [41], 16, 0)]  # more slots than are cut


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", MANY, ids=lambda c: str(c)[:60])
def test_many_tiles_and_many_sequences(gpu, dtype, case):
    from kuiperllama_amd import ops
    H, KH, D, DV, new, lens, page, window = case
    gen = generator(len(lens) + D)
    kc, vc, table, ks, vs = paged(gen, dtype, KH, D, DV, lens, page)
    T = sum(new)
    q = rnd(gen, dtype, T + 1, H, D, scale=1.5)
    lengths = torch.tensor(lens, dtype=torch.int32, device=gpu)
    ws = ops.attn_paged_workspace(H, KH, DV, T + 1, gpu)
    for max_new in (None, max(new)) if max(new) < 32 else (None,):
        out = torch.full((T + 1, H, DV), 9.0, dtype=dtype, device=gpu)
        ops.attn_paged(q, kc, vc, table, lengths, offsets_of(new, gpu), out, ws, window=window, max_new=max_new)
        check_paged(q, out, lens, new, ks, vs, window, f"max_new {max_new}")
        assert (out[T:] == 9.0).all()
    assert not ws[:4096].any()
