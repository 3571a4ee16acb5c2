"""Operators over many tokens of several sequences (ops.rope_tokens, rope_store, attn_packed, attn_paged): what they refuse, and the
table of angles, without a GPU."""
import ctypes as C
import math

import pytest
import torch

from kuiperllama_amd import _ffi, build, ops

P = 4096  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    build.build_lib()
    return _ffi.lib()


def rope_rows(**kw):
    r = dict(dtype=1, mode=1, n_tokens=4, head_num=4, kv_head_num=2, head_size=64, rot_dim=64, magnitude=1.0, turns=P, positions=P, q=P, k=P,
             q_token=256, q_head=64, k_token=128, k_head=64, q_out=P, k_out=P, qo_token=256, qo_head=64, ko_token=128, ko_head=64)
    r.update(kw)
    return _ffi.RopeRows(**r)


def cache(**kw):
    c = dict(k=P, v=P, k_page=2048, k_slot=128, k_head=64, v_page=2048, v_slot=128, v_head=64, n_pages=8, page_size=16)
    c.update(kw)
    return _ffi.PageCache(**c)


def attn_rows(**kw):
    r = dict(dtype=1, n_tokens=4, n_seqs=2, head_num=4, kv_head_num=2, head_size=64, value_size=64, window=0, scale=0.125, offsets=P, q=P,
             q_token=256, q_head=64, out=2 * P, o_token=256, o_head=64)
    r.update(kw)
    return _ffi.AttnRows(**r)


ROWS_REFUSED = [dict(dtype=0), dict(dtype=3), dict(mode=2), dict(n_tokens=-1), dict(head_num=0), dict(kv_head_num=3), dict(rot_dim=63), dict(rot_dim=66),
                dict(rot_dim=-2), dict(magnitude=math.inf), dict(magnitude=math.nan), dict(turns=None), dict(positions=None), dict(q=None), dict(k=P + 8),
                dict(q_out=None), dict(q_token=252), dict(k_head=68), dict(qo_head=4), dict(head_size=0)]


@pytest.mark.parametrize("bad", ROWS_REFUSED + [dict(k_out=None), dict(ko_token=130)], ids=str)
def test_rope_tokens_refuses(lib, bad):
    assert lib.kh_rope_tokens(C.byref(rope_rows(**bad)), None) == -1


@pytest.mark.parametrize("bad", ROWS_REFUSED, ids=str)
def test_rope_store_refuses_rows(lib, bad):
    assert lib.kh_rope_store(C.byref(rope_rows(**bad)), P, 128, 64, 64, C.byref(cache()), P, None) == -1


def test_rope_store_refuses_caches(lib):
    r = C.byref(rope_rows())
    for bad in (dict(k=None), dict(v=P + 4), dict(n_pages=0), dict(page_size=0), dict(k_page=2044), dict(k_slot=4), dict(v_head=65), dict(v_page=1)):
        assert lib.kh_rope_store(r, P, 128, 64, 64, C.byref(cache(**bad)), P, None) == -1, bad
    c = C.byref(cache())
    assert lib.kh_rope_store(r, None, 128, 64, 64, c, P, None) == -1
    assert lib.kh_rope_store(r, P, 128, 64, 0, c, P, None) == -1
    assert lib.kh_rope_store(r, P, 128, 64, 64, c, None, None) == -1
    assert lib.kh_rope_store(r, P, 130, 64, 64, c, P, None) == -1
    assert lib.kh_rope_store(r, P, 128, 64, 64, None, P, None) == -1


def test_sizes_that_are_not_supported(lib):
    assert lib.kh_rope_tokens(C.byref(rope_rows(head_size=264, rot_dim=8)), None) == _ffi.KH_ERR_UNSUPPORTED
    assert lib.kh_rope_tokens(C.byref(rope_rows(head_size=60, rot_dim=8)), None) == _ffi.KH_ERR_UNSUPPORTED
    assert lib.kh_rope_store(C.byref(rope_rows()), P, 128, 64, 60, C.byref(cache()), P, None) == _ffi.KH_ERR_UNSUPPORTED
    for kw in (dict(head_size=264), dict(value_size=264), dict(head_size=60), dict(value_size=4), dict(dtype=2, head_size=66),
               dict(n_tokens=1 << 30), dict(n_seqs=1 << 30)):
        assert lib.kh_attn_packed(C.byref(attn_rows(**kw)), P, 128, 64, P, 128, 64, None) == _ffi.KH_ERR_UNSUPPORTED, kw


ATTN_REFUSED = [dict(dtype=0), dict(dtype=3), dict(n_tokens=-1), dict(n_seqs=-1), dict(head_num=0), dict(kv_head_num=3), dict(head_size=0),
                dict(value_size=-8), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(offsets=None), dict(q=None),
                dict(q=P + 8), dict(out=None), dict(q_token=252), dict(o_head=68)]


@pytest.mark.parametrize("bad", ATTN_REFUSED, ids=str)
def test_attention_refuses_rows(lib, bad):
    r = C.byref(attn_rows(**bad))
    assert lib.kh_attn_packed(r, P, 128, 64, P, 128, 64, None) == -1
    assert lib.kh_attn_paged(r, C.byref(cache()), P, 4, 4, P, 0, P, 1 << 40, None) == -1


def test_attention_refuses_keys(lib):
    r = C.byref(attn_rows())
    for a in ((None, 128, 64, P, 128, 64), (P, 128, 64, None, 128, 64), (P + 2, 128, 64, P, 128, 64), (P, 129, 64, P, 128, 64), (P, 128, 64, P, 128, 63)):
        assert lib.kh_attn_packed(r, *a, None) == -1, a
    c = C.byref(cache())
    ok = [r, c, P, 4, 4, P, 0, P, 1 << 40, None]
    for at, value in ((1, None), (2, None), (3, -1), (4, 0), (5, None), (6, -1), (7, None), (7, P + 8), (8, 0)):
        a = list(ok)
        a[at] = value
        assert lib.kh_attn_paged(*a) == -1, (at, value)
    for bad in (dict(k=None), dict(v=P + 4), dict(n_pages=0), dict(page_size=0), dict(page_size=(1 << 20) + 1), dict(k_page=2044), dict(v_slot=4)):
        assert lib.kh_attn_paged(r, C.byref(cache(**bad)), P, 4, 4, P, 0, P, 1 << 40, None) == -1, bad


def test_nothing_to_do_is_no_error(lib):
    assert lib.kh_rope_tokens(C.byref(rope_rows(n_tokens=0)), None) == 0
    assert lib.kh_rope_store(C.byref(rope_rows(n_tokens=0)), P, 128, 64, 64, C.byref(cache()), P, None) == 0
    for kw in (dict(n_tokens=0), dict(n_seqs=0)):
        assert lib.kh_attn_packed(C.byref(attn_rows(**kw)), P, 128, 64, P, 128, 64, None) == 0
        assert lib.kh_attn_paged(C.byref(attn_rows(**kw)), C.byref(cache()), P, 4, 4, P, 0, P, 1 << 40, None) == 0


def test_nothing_to_do_needs_no_addresses(lib):
    """An empty tensor has none."""
    none = dict(turns=None, positions=None, q=None, k=None, q_out=None)
    assert lib.kh_rope_tokens(C.byref(rope_rows(n_tokens=0, k_out=None, **none)), None) == 0
    assert lib.kh_rope_store(C.byref(rope_rows(n_tokens=0, **none)), None, 128, 64, 64, C.byref(cache()), None, None) == 0
    r = C.byref(attn_rows(n_tokens=0, q=None, out=None, offsets=None))
    assert lib.kh_attn_packed(r, None, 128, 64, None, 128, 64, None) == 0
    assert lib.kh_attn_paged(r, C.byref(cache()), None, 4, 4, None, 0, None, 0, None) == 0


def test_places_that_overlap_are_refused(lib):
    """Results where rows are still to be read: in place with other strides, an output that is the queries."""
    other = P + 4096
    for at, to in (("q_token", "qo_token"), ("q_head", "qo_head"), ("k_token", "ko_token"), ("k_head", "ko_head")):
        r = rope_rows(**{to: 8 * getattr(rope_rows(), at)})
        assert lib.kh_rope_tokens(C.byref(r), None) == -1, at
        if at[0] == "q":
            assert lib.kh_rope_store(C.byref(r), P, 128, 64, 64, C.byref(cache()), P, None) == -1, at
    r = C.byref(attn_rows(out=P))  # q too
    assert lib.kh_attn_packed(r, other, 128, 64, other, 128, 64, None) == -1
    assert lib.kh_attn_paged(r, C.byref(cache()), P, 4, 4, P, 0, P, 1 << 40, None) == -1


def test_launches_that_no_grid_holds(lib):
    assert lib.kh_rope_tokens(C.byref(rope_rows(n_tokens=1 << 24)), None) == _ffi.KH_ERR_UNSUPPORTED
    assert lib.kh_rope_store(C.byref(rope_rows(n_tokens=1 << 24)), P, 128, 64, 64, C.byref(cache()), P, None) == _ffi.KH_ERR_UNSUPPORTED
    for kw in (dict(n_seqs=1 << 23), dict(n_tokens=1 << 28)):
        assert lib.kh_attn_packed(C.byref(attn_rows(**kw)), P, 128, 64, P, 128, 64, None) == _ffi.KH_ERR_UNSUPPORTED, kw


def test_workspace_sizes(lib):
    for bad in ((0, 1, 64, 1), (4, 3, 64, 1), (4, 2, 0, 1), (4, 2, 64, -1)):
        assert lib.kh_attn_paged_workspace_bytes(*bad) == -1, bad
    assert 0 < lib.kh_attn_paged_workspace_bytes(32, 8, 128, 64) < 1 << 30
    with pytest.raises(_ffi.KhError):
        ops.attn_paged_workspace(4, 3, 64, 1, "cpu")


def test_host_tensors_are_refused():
    t, i = torch.zeros(4, 2, 64), torch.zeros(4, dtype=torch.int32)
    table = ops.rope_table(64, 1e4, "cpu")
    c = torch.zeros(2, 16, 2, 64)
    for call in (lambda: ops.rope_tokens(t, t, i, table, 1), lambda: ops.rope_store(t, t, t, i, table, 1, c, c, i),
                 lambda: ops.attn_packed(t, t, t, i, t), lambda: ops.attn_paged(t, c, c, i[None], i[:1], i[:2], t, i.to(torch.uint8))):
        with pytest.raises(ValueError, match="GPU"):
            call()


# ---- the table of angles ---------------------------------------------------------------------------------------------
def frequencies(rot, theta, scaling):
    """Radians a position, one pair at a time, and the factor."""
    out, factor = [], 1.0
    for i in range(rot // 2):
        f = theta ** (-2.0 * i / rot)
        kind = (scaling or {}).get("rope_type")
        if kind == "linear":
            f /= scaling["factor"]
        elif kind == "llama3":
            wave, old = 2 * math.pi / f, scaling["original_max_position_embeddings"]
            if wave > old / scaling["low_freq_factor"]:
                f /= scaling["factor"]
            elif wave >= old / scaling["high_freq_factor"]:
                mix = (old / wave - scaling["low_freq_factor"]) / (scaling["high_freq_factor"] - scaling["low_freq_factor"])
                f = (1 - mix) * f / scaling["factor"] + mix * f
        elif kind == "yarn":
            at = [rot * math.log(scaling["original_max_position_embeddings"] / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in
                  (scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0))]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
            mix = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = mix * f / scaling["factor"] + (1 - mix) * f
            factor = scaling.get("attention_factor") or 0.1 * math.log(scaling["factor"]) + 1.0
        out.append(f)
    return out, factor


SCALINGS = [None, {"rope_type": "default"}, {"rope_type": "linear", "factor": 4.0},
            {"rope_type": "llama3", "factor": 32.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192},
            {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096},
            {"rope_type": "yarn", "factor": 2.0, "beta_fast": 16.0, "beta_slow": 2.0, "original_max_position_embeddings": 100, "attention_factor": 0.7}]


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: str((s or {}).get("rope_type")))
@pytest.mark.parametrize("rot,theta", [(128, 10000.0), (64, 500000.0), (2, 10000.0), (20, 1e6)])
def test_turns(rot, theta, scaling):
    turns, magnitude = ops.rope_turns(rot, theta, scaling)
    want, factor = frequencies(rot, theta, scaling)
    assert len(turns) == rot // 2 and magnitude == pytest.approx(factor, rel=2 ** -23)
    for t, f in zip(turns, want):
        # a few roundings of 64 bits each side: pow, products, the quotient by 2 pi
        assert abs(t / 2 ** 64 - f / (2 * math.pi) % 1.0) <= 16 * 2 ** -53 * f / (2 * math.pi) + 2 ** -64


def test_yarn_s_factor():
    """Of the two factors of a model with latent keys; 1 where nothing is stretched; refused where the borders are no pairs."""
    yarn = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}
    factor = lambda **kw: ops.rope_turns(64, 1e4, {**yarn, **kw})[1]  # noqa: E731
    assert factor(mscale=0.707, mscale_all_dim=1.0) == pytest.approx((0.0707 * math.log(40) + 1) / (0.1 * math.log(40) + 1), rel=2 ** -23)
    assert factor(mscale=1.0, mscale_all_dim=1.0) == 1.0
    assert factor(mscale=0.707) == factor(attention_factor=None) == pytest.approx(0.1 * math.log(40) + 1, rel=2 ** -23)
    assert factor(mscale=0.5, mscale_all_dim=1.0, attention_factor=1.5) == 1.5
    assert factor(factor=0.5) == 1.0
    with pytest.raises(ValueError, match="truncate"):
        factor(truncate=False)
    with pytest.raises(KeyError, match="original_max_position_embeddings"):
        ops.rope_turns(64, 1e4, {"rope_type": "yarn", "factor": 40.0})


def test_turns_refuse(lib):
    u, m = (C.c_uint64 * 64)(), C.c_float()
    S = _ffi.RopeScaling
    for rot, theta, s in ((63, 1e4, None), (-2, 1e4, None), (258, 1e4, None), (64, 0.0, None), (64, -1.0, None), (64, math.nan, None), (64, math.inf, None),
                          (64, 1e4, S(kind=4)), (64, 1e4, S(kind=-1)), (64, 1e4, S(kind=1, factor=0.0)), (64, 1e4, S(kind=1, factor=math.nan)),
                          (64, 1e4, S(kind=2, factor=2.0, original=8.0, low=4.0, high=4.0)), (64, 1e4, S(kind=2, factor=2.0, original=0.0, low=1.0, high=4.0)),
                          (64, 1e4, S(kind=3, factor=2.0, original=8.0, fast=1.0, slow=1.0)), (64, 1.0, S(kind=3, factor=2.0, original=8.0, fast=32.0, slow=1.0)),
                          (64, 1e4, S(kind=3, factor=2.0, original=8.0, fast=32.0, slow=1.0, magnitude=-1.0))):
        assert lib.kh_rope_turns(rot, theta, C.byref(s) if s is not None else None, u, C.byref(m)) == -1, (rot, theta)
    assert lib.kh_rope_turns(64, 1e4, None, None, C.byref(m)) == -1
    assert lib.kh_rope_turns(64, 1e4, None, u, None) == -1
    assert lib.kh_rope_turns(0, 1e4, None, None, C.byref(m)) == 0 and m.value == 1.0
    with pytest.raises(ValueError, match="rope_type"):
        ops.rope_turns(64, 1e4, {"rope_type": "other"})
    with pytest.raises(KeyError):
        ops.rope_turns(64, 1e4, {"rope_type": "linear"})


def test_pages_of_every_size_divide_exactly():
    """The multiplier that the attention divides places by: floor((2^(31+b)) / d) + 1, its high word shifted by b - 1."""
    for d in list(range(2, 600)) + [1000, 1023, 1024, 1025, 65535, 65536, 65537, (1 << 20) - 1, 1 << 20]:
        b = (d - 1).bit_length()
        magic = (1 << (31 + b)) // d + 1
        assert magic < 1 << 32
        for q in (0, 1, 2, 3, 1000, (2 ** 31 - 1) // d - 1, (2 ** 31 - 1) // d):
            for n in (q * d - 1, q * d, q * d + 1):
                if 0 <= n < 2 ** 31:
                    assert ((n * magic) >> 32) >> (b - 1) == n // d, (d, n)


def test_outputs_whose_rows_lie_in_one_another_are_refused(lib):
    """An expanded tensor, or strides shorter than what lies within them: several workgroups would write one place, and a rotation in place
    would turn a row that heads share once a head.  Of one row a stride says nothing."""
    packed = lambda k=3 * P, v=4 * P, **kw: lib.kh_attn_packed(C.byref(attn_rows(**kw)), k, 128, 64, v, 128, 64, None)  # noqa: E731
    paged = lambda c=cache(k=3 * P, v=4 * P), **kw: lib.kh_attn_paged(C.byref(attn_rows(**kw)), C.byref(c), P, 4, 4, P, 0, P, 1 << 40, None)  # noqa: E731
    apart = dict(q_out=2 * P, k_out=3 * P)
    tokens = lambda **kw: lib.kh_rope_tokens(C.byref(rope_rows(**{**apart, **kw})), None)  # noqa: E731
    store = lambda c=cache(v=3 * P), **kw: lib.kh_rope_store(C.byref(rope_rows(**{**apart, **kw})), P, 128, 64, 64, C.byref(c), P, None)  # noqa: E731
    for token, head in ((0, 64), (256, 0), (0, 0), (192, 64), (256, 56), (64, 64), (-192, 64), (64, 128)):
        for call in (packed, paged):
            assert call(o_token=token, o_head=head) == -1, (token, head)
        for call in (tokens, store):
            assert call(qo_token=token, qo_head=head) == -1, (token, head)
    for token, head in ((0, 64), (128, 0), (64, 64)):
        assert tokens(ko_token=token, ko_head=head) == -1, (token, head)
        assert tokens(k_out=P, k_token=token, k_head=head, ko_token=token, ko_head=head) == -1, "in place"
    for bad in (dict(k_page=0), dict(k_slot=0), dict(k_head=0), dict(v_page=1984), dict(v_slot=64), dict(v_head=8)):
        assert store(c=cache(**{"v": 3 * P, **bad})) == -1, bad
    # one place for two results, a result where keys or values are still to be read
    assert tokens(k_out=2 * P) == -1
    assert store(c=cache()) == -1  # k and v
    assert packed(k=2 * P) == -1 and packed(v=2 * P) == -1
    assert paged(c=cache(k=2 * P, v=4 * P)) == -1 and paged(c=cache(k=3 * P, v=2 * P)) == -1


def test_turns_that_are_no_numbers_are_refused(lib):
    """Frequencies and factors beyond what a number holds: there is no fraction of a turn to give."""
    u, m = (C.c_uint64 * 128)(), C.c_float()
    S = _ffi.RopeScaling
    for theta, s in ((1e-299, S(kind=1, factor=1e-299)), (1e4, S(kind=1, factor=5e-324)), (1e4, S(kind=2, factor=5e-324, original=8192.0, low=1.0, high=4.0)),
                     (1e4, S(kind=2, factor=8.0, original=math.inf, low=1.0, high=math.inf)),
                     (1e4, S(kind=3, factor=5e-324, original=4096.0, fast=32.0, slow=1.0)),
                     (1e4, S(kind=3, factor=8.0, original=4096.0, fast=32.0, slow=1.0, magnitude=math.inf)),
                     (1e4, S(kind=3, factor=8.0, original=4096.0, fast=32.0, slow=1.0, magnitude=1e39))):
        assert lib.kh_rope_turns(256, theta, C.byref(s), u, C.byref(m)) == -1, (theta, s.kind)
    assert lib.kh_rope_turns(256, 1e-299, None, u, C.byref(m)) == 0  # the fastest pair: 1e296 radians a position, and a number


def test_scales_that_have_no_room_in_base_two_are_refused(lib):
    """Exponentials run in base two: scale log2 e has to be a number too."""
    for scale in (2.37e38, 3.4e38):
        r = C.byref(attn_rows(scale=scale))
        assert lib.kh_attn_packed(r, 3 * P, 128, 64, 4 * P, 128, 64, None) == -1, scale
        assert lib.kh_attn_paged(r, C.byref(cache(k=3 * P, v=4 * P)), P, 4, 4, P, 0, P, 1 << 40, None) == -1, scale
