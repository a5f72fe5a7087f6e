"""Refusals of the paged key-value cache entry points.  Arguments are checked
before a device is touched, so these run without a GPU: a refused call answers
INVALID and names the fault, a sound one gets as far as the missing device."""
import pytest

torch = pytest.importorskip("torch")

from krikil_rs_b200 import _lib, kernels as K  # noqa: E402
from krikil_rs_b200._lib import lib  # noqa: E402

P = 4096  # a placeholder address, aligned to 16 bytes: never read

PLAN = dict(new=P, lens=P, table=P, ld=8, B=2, width=8, free=P, count=P, num_pages=64, page=16, lens_out=P,
            count_out=P, cu=P, positions=P, slots=P, rows=4, status=P, stream=None)
RELEASE = dict(done=P, lens=P, table=P, ld=8, B=2, width=8, free=P, count=P, num_pages=64, page=16, lens_out=P,
               count_out=P, status=P, stream=None)
APPEND = dict(q=P, q_st=512, q_sh=64, k=P, k_st=128, k_sh=64, v=P, v_st=128, v_sh=64, type=0, qo=P, qo_st=512,
              qo_sh=64, kc=P, vc=P, c_sp=2048, c_st=128, c_sh=64, ctype=0, slots=P, positions=P, T=3, Hq=8, Hkv=2,
              dh=64, rot=64, num_pages=64, page=16, theta=10000.0, stream=None)
ATTN = dict(q=P, q_sb=512, q_sh=64, type=0, kc=P, vc=P, c_sp=2048, c_st=128, c_sh=64, ctype=0, table=P, ld=8, width=8,
            num_pages=64, page=16, lens=P, B=3, Hq=8, Hkv=2, dh=64, scale=0.125, window=0, max_len=0, out=P, o_sb=512,
            o_sh=64, lse=P, work=P, work_floats=1 << 40, stream=None)

POOL = [("page", 0, "power of two"), ("page", 12, "power of two"), ("page", 131072, "power of two"),
        ("num_pages", 0, "num_pages"), ("num_pages", -3, "num_pages"), ("num_pages", 1 << 27, "num_pages")]
TABLE = [("width", 0, "width"), ("width", 1 << 28, "width"), ("ld", 7, "table_ld")]
TYPES = [("type", 3, "type"), ("ctype", -1, "type"), (("type", "ctype"), (1, 2), "16-bit q"),
         (("type", "ctype"), (2, 0), "16-bit q")]
HEAD = [("dh", 0, "dh"), ("dh", 66, "dh"), ("dh", 260, "dh")]


def refused(fn, base, what, value, word):
    args = dict(base)
    if isinstance(what, tuple):
        args.update(zip(what, value))
    else:
        args[what] = value
    assert list(args) == list(base)
    assert fn(*args.values()) == _lib.INVALID, (what, value)
    assert word in lib.krk_last_error().decode(), lib.krk_last_error()


@pytest.mark.parametrize("what,value,word", POOL + TABLE + [("B", 0, "B must"), ("B", -1, "B must"),
                                                            ("rows", -1, "rows")]
                         + [(n, None, "null") for n in ("new", "lens", "table", "free", "count", "lens_out",
                                                        "count_out", "cu", "positions", "slots", "status")])
def test_page_plan_refuses(what, value, word):
    refused(lib.krk_k_kv_page_plan, PLAN, what, value, word)


@pytest.mark.parametrize("what,value,word", POOL + TABLE + [("B", 0, "B must")]
                         + [(n, None, "null") for n in ("done", "lens", "table", "free", "count", "lens_out",
                                                        "count_out", "status")])
def test_page_release_refuses(what, value, word):
    refused(lib.krk_k_kv_page_release, RELEASE, what, value, word)


@pytest.mark.parametrize("what,value,word", POOL + TYPES + HEAD + [
    ("T", -1, "T and"), ("Hq", -1, "Hq"), ("Hkv", 0, "Hkv"), ("Hq", 65536, "heads"),
    ("rot", -2, "rot_dim"), ("rot", 65, "rot_dim"), ("rot", 66, "rot_dim"),
    ("theta", 0.0, "theta"), ("theta", -1.0, "theta"), ("theta", float("nan"), "theta"),
    ("theta", float("inf"), "theta"), ("slots", None, "null"), ("positions", None, "null"),
    ("c_st", 60, "shorter"), ("c_sp", 0, "shorter"), ("c_sh", 32, "shorter"), ("qo_st", 0, "shorter")]
    + [(n, None, "pointers") for n in ("q", "k", "v", "qo", "kc", "vc")]
    + [(n, P + 8, "aligned") for n in ("q", "k", "v", "qo", "kc", "vc")]
    + [(n, 513, "multiples of four") for n in ("q_st", "q_sh", "k_st", "k_sh", "v_st", "v_sh", "qo_st", "qo_sh",
                                               "c_sp", "c_st", "c_sh")]
    + [("k_st", -512, "multiples of four")])
def test_append_refuses(what, value, word):
    refused(lib.krk_k_rope_kv_append_paged, APPEND, what, value, word)


@pytest.mark.parametrize("what,value,word", POOL + TABLE + TYPES + HEAD + [
    ("B", -1, "B must"), ("B", 1 << 30, "B * Hq"), ("Hq", 0, "Hq"), ("Hkv", 0, "Hkv"), ("Hq", 7, "multiple"), ("Hq", 65536, "65535"),
    ("scale", float("nan"), "scale"), ("scale", float("inf"), "scale"), ("window", -1, "window"),
    ("max_len", -1, "max_len"), ("table", None, "null"), ("lens", None, "null"),
    ("o_sb", 0, "shorter"), ("o_sh", 32, "shorter")]
    + [(n, None, "pointers") for n in ("q", "kc", "vc", "out")]
    + [(n, P + 8, "aligned") for n in ("q", "kc", "vc", "out")]
    + [(n, 514, "multiples of four") for n in ("q_sb", "q_sh", "c_sp", "c_st", "c_sh", "o_sb", "o_sh")])
def test_attention_refuses(what, value, word):
    refused(lib.krk_k_attn_decode_paged, ATTN, what, value, word)


def test_half_precision_pointers_need_eight_bytes_only():
    """Four 16-bit elements: an address that is a multiple of 8 passes the checks where one of 4 does not."""
    half = dict(ATTN, type=1, ctype=1)
    refused(lib.krk_k_attn_decode_paged, half, "q", P + 4, "aligned")
    if not torch.cuda.is_available():
        assert lib.krk_k_attn_decode_paged(*dict(half, q=P + 8).values()) == _lib.CUDA


def test_empty_steps_are_done_at_once():
    assert lib.krk_k_rope_kv_append_paged(*dict(APPEND, T=0, q=None, k=None, v=None, slots=None).values()) == _lib.OK
    assert lib.krk_k_attn_decode_paged(*dict(ATTN, B=0, q=None, table=None, lens=None, out=None).values()) == _lib.OK


def test_sizes_of_the_attention_scratch():
    f = lib.krk_attn_paged_work_floats
    assert f(4, 8, 8, 64, 100000, 0) > 0
    assert f(4, 8, 8, 64, 1, 0) == 0 and f(4, 8, 8, 64, 100000, 100) == 0  # few keys need none
    for bad in ((0, 8, 8, 64, 9999, 0), (4, 8, 3, 64, 9999, 0), (4, 8, 8, 62, 9999, 0), (4, 0, 1, 64, 9999, 0),
                (4, 8, 0, 64, 9999, 0), (4, 8, 8, 64, -1, 0), (4, 8, 8, 64, 9999, -1)):
        assert f(*bad) == 0


def clusters(items, units, sms):
    """Whether a launch of so many pieces of so many 64-key units takes clusters, which need no scratch (shares do):
    up to 8 blocks a piece in a wave of three a multiprocessor, 24 units a block, 8 when the device is not full."""
    if items > 3 * sms:
        return False
    n = 1
    while n < 8 and units > 2 * n and items * 2 * n <= 3 * sms:
        n *= 2
    return units <= (24 if items * n >= sms else 8) * n


def pieces(g, heads):
    """Of a cache head with g query heads, `heads` of them a warp, 1, 2 or 4 warps side by side."""
    groups = 1 if g <= heads else 2 if g <= 2 * heads else 4
    return -(-g // (groups * heads))


def test_scratch_for_every_launch_that_takes_shares():
    """The types are not known to the size of the scratch, and engines differ in their pieces: whichever takes shares
    must have got some."""
    f = lib.krk_attn_paged_work_floats
    sms = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148
    bounds = [1, 64, 65, 128, 129, 500, 1000, 1500, 2048, 3000, 4096, 4097, 5000, 6144, 6145, 8000, 8192, 10000, 12288,
              12289, 16000, 20000, 24576, 32768]
    for g in range(1, 129):
        engines = {1 if g == 1 else 2 if g == 2 else 4, 8}
        for heads in [*range(1, 160), 161, 199, 222, 223, 296, 297, 444, 445, 500]:  # B * Hkv
            for n in bounds:
                if not all(clusters(heads * pieces(g, e), -(-n // 64), sms) for e in engines):
                    assert f(heads, g, 1, 64, n, 0) > 0, (g, heads, n)


@pytest.mark.parametrize("b,hq,hkv,dh,n,window", [(10, 32, 1, 64, 8192, 0), (10, 32, 1, 128, 8000, 0),
                                                  (5, 64, 2, 64, 4097, 0), (8, 48, 1, 128, 100000, 6000),
                                                  (4, 71, 1, 64, 12000, 0), (3, 128, 1, 64, 12288, 0)])
def test_scratch_for_many_heads_on_one_cache_head(b, hq, hkv, dh, n, window):
    assert lib.krk_attn_paged_work_floats(b, hq, hkv, dh, n, window) > 0


def test_table_rows_that_lie_closer_than_their_width_are_refused():
    """A row expanded over the requests, or a sliding view: rows must not be taken to lie `width` apart."""
    cpu = torch.device("cpu")
    row = torch.arange(6, dtype=torch.int32)
    for bad in (row[None].expand(3, 6), row.as_strided((3, 4), (1, 1)), row[:1].expand(2, 1)):
        with pytest.raises(ValueError, match="table"):
            K._table(bad, cpu)
    assert K._table(row[None], cpu) == (1, 6, 6) and K._table(row.expand(1, 6), cpu) == (1, 6, 6)
    assert K._table(row.as_strided((1, 6), (0, 1)), cpu) == (1, 6, 6)  # one row: its stride does not matter
    assert K._table(torch.zeros(3, 9, dtype=torch.int32)[:, 2:7], cpu) == (3, 5, 9)
    assert K._table(row[None][:0], cpu) == (0, 6, 6)


def test_wrappers_refuse_cpu_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 2, 64)
    pool = torch.zeros(4, 16, 2, 64)
    table = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        K.kv_page_plan(i, i, table, i, i[:1], 16, 4)
    with pytest.raises(ValueError, match="CUDA"):
        K.kv_page_release(i.bool(), i, table, i, i[:1], 16)
    with pytest.raises(ValueError, match="CUDA"):
        K.rope_kv_append_paged(x, x, x, pool, pool, i, i)
    with pytest.raises(ValueError, match="CUDA"):
        K.attn_decode_paged(x, pool, pool, table, i)


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38])
def test_a_scale_that_leaves_32_bits_in_base_two_is_refused(scale):
    """Scores are taken times log2(e): such a scale would make NaN of a score of 0."""
    refused(lib.krk_k_attn_decode_paged, ATTN, "scale", scale, "scale")
