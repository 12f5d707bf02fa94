"""What the operators of 8-bit codes refuse, and their plain forms (no GPU)."""
import pytest
import torch

import int8_plain as plain

I8, F32, BF16, I32 = torch.int8, torch.float32, torch.bfloat16, torch.int32


def empty(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype)


def store_args(**change):
    a = dict(qkv=empty(5, 5 * 64, dtype=BF16), q=empty(5, 3 * 64, dtype=BF16), pos=empty(5, dtype=I32), seq=empty(5, dtype=I32),
             table=empty(2, 3, dtype=I32), cos=empty(9, 32), sin=empty(9, 32), k=empty(4, 1, 64, 64, dtype=I8), v=empty(4, 1, 64, 64, dtype=I8),
             ks=empty(4, 1, 64), vs=empty(4, 1, 64), heads=3, kv_heads=1, d=64, page=64)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,why", [
    (dict(), "CUDA tensors only"), (dict(qkv=empty(5, 5 * 64, dtype=torch.float16)), "float16"), (dict(q=empty(5, 3 * 64)), "q is"),
    (dict(q=empty(4, 3 * 64, dtype=BF16)), "q is"), (dict(k=empty(4, 1, 64, 64)), "k is"), (dict(v=empty(3, 1, 64, 64, dtype=I8)), "v is"),
    (dict(ks=empty(4, 1, 63)), "k_scales is"), (dict(vs=empty(4, 1, 64, dtype=BF16)), "v_scales is"), (dict(pos=empty(4, dtype=I32)), "each of 5 rows"),
    (dict(seq=empty(5, dtype=torch.int64)), "token_seq is"), (dict(table=empty(6, dtype=I32)), "page_table is"), (dict(sin=None), "cos and sin"),
    (dict(cos=empty(9, 31)), "cos is"), (dict(sin=empty(8, 32)), "sin is"), (dict(heads=0), "query head"), (dict(d=63), "even head sizes"),
    (dict(kv_heads=0), "even head sizes"), (dict(qkv=empty(5, 6 * 64, dtype=BF16)[:, 64:]), "not contiguous")])
def test_writing_refuses(change, why):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match=why):
        ops.rope_store_int8(*store_args(**change))


def read_args(**change):
    a = dict(k=empty(4, 2, 64, 64, dtype=I8), v=empty(4, 2, 64, 64, dtype=I8), ks=empty(4, 2, 64), vs=empty(4, 2, 64), table=empty(2, 3, dtype=I32),
             local=empty(2, 3, dtype=I32), ko=empty(5, 2, 64, 64, dtype=BF16), vo=empty(5, 2, 64, 64, dtype=BF16))
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,why", [
    (dict(), "CUDA tensors only"), (dict(k=empty(4, 2, 64, 64)), "k is"), (dict(k=empty(4, 64, 64, dtype=I8)), "k is int8"),
    (dict(vs=empty(4, 64, 2)), "v_scales is"), (dict(local=empty(2, 3, dtype=torch.int64)), "local_table is"), (dict(vo=empty(5, 2, 64, 64)), "v_out is"),
    (dict(ko=empty(5, 2, 64, 63, dtype=BF16)), "k_out is"), (dict(vo=empty(4, 2, 64, 64, dtype=BF16)), "v_out is"),
    (dict(ko=empty(5, 2, 64, 64, dtype=torch.float16)), "float16")])
def test_reading_refuses(change, why):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match=why):
        ops.read_pages_int8(*read_args(**change))


def attend_args(**change):
    a = dict(q=empty(5, 6 * 64, dtype=BF16), stride=6 * 64, k=empty(4, 2, 64, 64, dtype=I8), v=empty(4, 2, 64, 64, dtype=I8), ks=empty(4, 2, 64),
             vs=empty(4, 2, 64), pos=empty(5, dtype=I32), seq=empty(5, dtype=I32), table=empty(2, 3, dtype=I32), out=empty(5, 6 * 64, dtype=BF16),
             heads=6, kv_heads=2, d=64, window=0, scale=0.125, ws=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,why", [
    (dict(), "CUDA tensors only"), (dict(q=empty(5, 6 * 64)), "out is"), (dict(out=empty(5, 5 * 64, dtype=BF16)), "out is"), (dict(k=empty(4, 2, 64, 64)), "k is"),
    (dict(ks=empty(4, 2, 64, 1)), "k_scales is"), (dict(pos=empty(5)), "token_pos is"), (dict(table=empty(2, 3)), "page_table is"),
    (dict(q=empty(5, 6 * 64, dtype=torch.float16), out=empty(5, 6 * 64, dtype=torch.float16)), "float16")])
def test_attention_refuses(change, why):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match=why):
        ops.attention_int8(*attend_args(**change))


def product_args(**change):
    a = dict(x=empty(5, 40, dtype=BF16), w=empty(12, 48, dtype=I8), ws=empty(12), bias=None, out=empty(5, 12, dtype=BF16), mode=0, space=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,why", [
    (dict(), "CUDA tensors only"), (dict(x=empty(5, 40, dtype=torch.float16)), "float16"), (dict(w=empty(12, 40, dtype=I8)), "w is"), (dict(w=empty(12, 48)), "w is"),
    (dict(ws=empty(11)), "w_scales is"), (dict(bias=empty(12, dtype=BF16)), "bias is"), (dict(out=empty(5, 12)), "out is"), (dict(mode=1), "out is"),
    (dict(mode=3), "out is"), (dict(mode=7), "mode 7"), (dict(w=empty(11, 48, dtype=I8), mode=3), "no gate and up")])
def test_products_refuse(change, why):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match=why):
        ops.linear_int8(*product_args(**change))


@pytest.mark.parametrize("x,codes,scales,why", [
    (empty(3, 20), empty(3, 32, dtype=I8), empty(3), "CUDA tensors only"), (empty(3, 20), empty(3, 20, dtype=I8), empty(3), "codes is"),
    (empty(3, 20), empty(3, 32, dtype=I8), empty(4), "scales is"), (empty(20, 3).T, empty(3, 32, dtype=I8), empty(3), "beside one another"),
    (empty(3, 0), empty(3, 0, dtype=I8), empty(3), "k >= 1"), (empty(3, 20, dtype=torch.float16), empty(3, 32, dtype=I8), empty(3), "float16")])
def test_codes_of_rows_refuse(x, codes, scales, why):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match=why):
        ops.quantize_rows(x, codes, scales)


def test_codes_are_within_half_a_step():
    x = torch.randn((200, 64), generator=torch.Generator().manual_seed(0))
    codes, scales = plain.codes_of(x)
    assert codes.abs().amax() == 127
    assert ((codes.double() * scales.double()[:, None] - x.double()).abs() <= x.abs().amax(1, keepdim=True).double() / 254 * (1 + 2.0 ** -20)).all()


def test_codes_of_bfloat16_rows_are_the_exact_quotients():
    """Every pair of a value and a top of 8 significant bits: the code is the exact quotient's, ties to even; half of the top, 63.5 steps,
    may go either way."""
    top = torch.arange(128, 256, dtype=F32)
    for e in (1.0, 0.5, 0.25, 2.0 ** -6):
        x = torch.arange(128, 256, dtype=F32) * e
        rows = torch.stack((x[None].expand(128, -1), top[:, None].expand(-1, 128)), -1)
        rows = rows[(x[None] <= top[:, None])]
        codes, _ = plain.codes_of(rows)
        whole = (rows[:, 0].double() * 127).div(rows[:, 1].double(), rounding_mode="floor")
        part = rows[:, 0].double() * 127 - whole * rows[:, 1].double()  # (exact)
        up = (2 * part > rows[:, 1]) | ((2 * part == rows[:, 1]) & (whole % 2 == 1))
        half = 2 * rows[:, 0] == rows[:, 1]
        assert torch.equal(codes[~half, 0].double(), (whole + up)[~half])
        assert ((codes[half, 0] == 63) | (codes[half, 0] == 64)).all()


# ---- the cache, the model and the command line --------------------------------------------------
def test_pages_of_codes_are_copied_with_their_scales():
    from nnis_b200.cache import CacheManager, KVRequest
    cache = CacheManager([KVRequest(2, 8, codes=True)] * 3 + [KVRequest(2, 8)], F32, torch.device("cpu"), 64 * 8, 4, 1000)
    codes, wide = cache.groups
    assert (codes.k.dtype, wide.k.dtype, codes.k_scales.shape, wide.k_scales) == (I8, F32, (3, 8, 2, 64), None)
    view = cache.view(1)
    assert view.k_scales.shape == (8, 2, 64) and view.v_scales.data_ptr() == codes.v_scales[1].data_ptr() and cache.view(3).k_scales is None
    a = cache.acquire()
    cache.reserve([a], [70])
    cache.commit([a], [70])
    for t in codes.stores():
        t[:, cache.page_table(0, a)[1], :, :6] = 9
    b = cache.fork(a)
    cache.reserve([b], [71])
    cache.commit([b], [71])
    mine, copy = cache.page_table(0, a)[1], cache.page_table(0, b)[1]
    assert mine != copy and all((t[:, copy, :, :6] == 9).all() and (t[:, copy, :, 6:] == 0).all() for t in codes.stores())
    assert cache.kv_bytes_per_token() == 3 * 2 * (16 + 8) + 2 * 16 * 4
    assert cache.kv_bytes_read(10) == 10 * cache.kv_bytes_per_token()
    assert cache.usage()["kv_bytes"] == 8 * 64 * cache.kv_bytes_per_token()
    cache.check()


def test_a_cache_of_codes_without_values_is_refused():
    from nnis_b200.cache import CacheManager, KVRequest
    with pytest.raises(ValueError, match="keys and values"):
        CacheManager([KVRequest(1, 8, values=False, codes=True)], F32, torch.device("cpu"), 64, 1, 64)


def test_models_without_an_8_bit_form_are_refused():
    import nafezen_models
    from helpers import TINY_A
    from nnis_b200.config import config_from_dict
    from nnis_b200.engine.model import DecoderModel
    cpu = torch.device("cpu")
    llama, other = config_from_dict(TINY_A).to_spec(), config_from_dict(nafezen_models.CONFIGS["mixed"]).to_spec()
    model = DecoderModel(llama, F32, cpu, "int8", "int8")
    assert all(r is None or r.codes for r in model.cache_requests())
    assert not any(r is not None and r.codes for r in DecoderModel(llama, F32, cpu).cache_requests())
    for args, why in ((("int8", None), "no 8-bit cache"), ((None, "int8"), "no 8-bit product")):
        with pytest.raises(ValueError, match=why):
            DecoderModel(other, F32, cpu, *args)
    for args in (("fp8", None), (None, "int4")):
        with pytest.raises(ValueError, match="must be None or 'int8'"):
            DecoderModel(llama, F32, cpu, *args)


def test_pages_that_a_prompt_step_reads_back():
    from nnis_b200.config import config_from_dict
    from nnis_b200.csrc import ops
    from nnis_b200.engine.model import DecoderModel
    from helpers import TINY_A
    spec = config_from_dict(TINY_A).to_spec()
    mixer = DecoderModel(spec, BF16, torch.device("cpu"), "int8").blocks[0].mixer
    few, many = ops.INT8_ROWS_AT_ONCE[BF16], ops.INT8_ROWS_AT_ONCE[BF16] + 1
    name = mixer._read_back_name()
    assert name not in mixer.step_tables([few, 1], [100, 0])
    tables = mixer.step_tables([1, many, 64], [100, 64, 0])
    assert tables[name].tolist() == [[0, 1], [2, 3], [4, -1]] and tables[name + "/pages"].tolist() == [5]
    assert name not in mixer.step_tables([many], [0], tuple(tables))  # (another layer has asked)
    mixer.window = 70
    assert mixer._read_back_table([many, 20], [200, 63])[0].tolist() == [[-1, -1, 0, 1], [2, 3, -1, -1]]


def test_flags_of_the_command_line():
    from nnis_b200.cli.main import UsageError, parse_args
    from nnis_b200.cli.process import ProcessContractError, execute
    base = ["generate", "--model", "m", "--prompt-ids", "1,2"]
    a = parse_args([*base, "--cache-dtype", "int8"])
    assert (a.cache_dtype, a.weight_dtype) == ("int8", None) and parse_args([*base, "--weight-dtype", "int8"]).weight_dtype == "int8"
    for flag in ("--cache-dtype", "--weight-dtype"):
        with pytest.raises(UsageError, match="must be int8"):
            parse_args([*base, flag, "float32"])
    with pytest.raises((ProcessContractError, ValueError)):
        execute("m", prompt_ids=[1], cache_dtype="fp8")


@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_plans_of_attention_cover_every_key(d):
    """Slices cover the table, clusters and tiles are what the kernel takes, and records fit a call's buffer."""
    from nnis_b200.csrc import ops
    for n, seqs in ((1, 1), (7, 7), (64, 64), (80, 16), (300, 300), (5, 400), (3000, 7)):
        for heads, kv_heads in ((9, 3), (32, 32), (20, 1), (64, 1), (16, 2)):
            for cols in (1, 2, 3, 63, 64, 500, 4096):
                for window in (0, 1, 64, 5000):
                    slices, pieces, rows, cluster, eights = ops.attention_int8_plan(n, seqs, heads, kv_heads, d, cols, window, 148)
                    per_page = 1 if d <= 64 else 2
                    assert 1 <= slices <= 64 and slices * pieces >= per_page * cols and (slices - 1) * pieces < per_page * cols
                    assert cluster in (0, 1, 2, 4, 8) and (cluster > 0 or slices == 1) and eights in (1, 2)
                    assert 1 <= rows <= max(1, 64 // (heads // kv_heads)) and slices * cluster <= 65535


def test_norms_and_coded_rows_refuse():
    from nnis_b200.csrc import ops
    x, w, codes, scales = empty(3, 20), empty(20), empty(3, 32, dtype=I8), empty(3)
    for args, why in (((x, w, 1e-5, codes, scales, BF16), "CUDA tensors only"), ((x, w, 0.0, codes, scales, BF16), "positive eps"),
                      ((empty(3, 21), empty(21), 1e-5, codes, scales, BF16), "multiple of 4"), ((x, empty(21), 1e-5, codes, scales, BF16), "weight is"),
                      ((x, w, 1e-5, empty(3, 20, dtype=I8), scales, BF16), "codes is"), ((x.to(BF16), w, 1e-5, codes, scales, BF16), "x is")):
        with pytest.raises(ops.KernelError, match=why):
            ops.rmsnorm_int8(*args)
    m, ms = empty(12, 32, dtype=I8), empty(12)
    for args, why in (((codes, scales, 20, m, ms, None, empty(3, 12), 0), "CUDA tensors only"), ((codes, scales, 40, m, ms, None, empty(3, 12), 0), "codes is"),
                      ((codes, empty(4), 20, m, ms, None, empty(3, 12), 0), "scales is"), ((codes, scales, 20, m, ms, empty(11), empty(3, 12), 0), "bias is"),
                      ((codes, scales, 20, m, ms, None, empty(3, 12), 3), "out is"), ((codes, scales, 20, m, ms, None, empty(3, 12, dtype=BF16), 1), "out is"),
                      ((codes, scales, 20, m, ms, None, empty(3, 12), 9), "mode 9")):
        with pytest.raises(ops.KernelError, match=why):
            ops.linear_int8_coded(*args)


@pytest.mark.parametrize("change,why", [
    (dict(window=1 << 31), "a window of 0 or more"), (dict(scale=float("inf")), "a positive scale"), (dict(scale=float("nan")), "a positive scale"),
    (dict(table=empty(2, 0, dtype=I32)), "at least one page"), (dict(table=empty(0, 3, dtype=I32)), "at least one page"),
    (dict(k=empty(0, 2, 64, 64, dtype=I8), v=empty(0, 2, 64, 64, dtype=I8), ks=empty(0, 2, 64), vs=empty(0, 2, 64)), "at least one page")])
def test_attention_without_a_page_or_a_scale_is_refused(change, why, monkeypatch):
    """(with the tensors taken for a GPU's: what is refused for where it lies is refused first)"""
    from nnis_b200.csrc import ops
    monkeypatch.setattr(ops, "_wanted", lambda what, **tensors: None)
    with pytest.raises(ops.KernelError, match=why):
        ops.attention_int8(*attend_args(**change))


@pytest.mark.parametrize("change", [dict(table=empty(2, 0, dtype=I32)),
                                    dict(k=empty(0, 1, 64, 64, dtype=I8), v=empty(0, 1, 64, 64, dtype=I8), ks=empty(0, 1, 64), vs=empty(0, 1, 64))])
def test_writing_without_a_page_is_refused(change):
    from nnis_b200.csrc import ops
    with pytest.raises(ops.KernelError, match="at least one page"):
        ops.rope_store_int8(*store_args(**change))


def test_operands_of_other_ranks_are_refused():
    from nnis_b200.csrc import ops
    for change in (dict(x=empty(5, 1, 40, dtype=BF16)), dict(x=empty(40, dtype=BF16)), dict(w=empty(48, dtype=I8))):
        with pytest.raises(ops.KernelError, match=r"x \[m, k\] and w"):
            ops.linear_int8(*product_args(**change))
    with pytest.raises(ops.KernelError, match=r"codes \[m, width\]"):
        ops.linear_int8_coded(empty(48, dtype=I8), empty(1), 40, empty(12, 48, dtype=I8), empty(12), None, empty(1, 12), ops.STORE)
    with pytest.raises(ops.KernelError, match=r"x \[n, width\]"):
        ops.rmsnorm_int8(empty(64), empty(64), 1e-5, empty(1, 64, dtype=I8), empty(1), BF16)
