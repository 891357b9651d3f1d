"""Rows of quantised tables by number: the bits of the dequantised rows times the factor, rounded once."""
import numpy as np
import pytest
import torch

from oracle import mxfp4_np as mx

gpu = pytest.mark.gpu


class Table:
    """A table of one of the three formats with its call and its dequantised rows."""

    def __init__(self, ops, synth, fmt, rows, n, seed):
        self.ops, self.fmt, self.rows, self.n = ops, fmt, rows, n
        if fmt == "mxfp4":
            codes, _s, tiles, _v = mx.random_matrix(rows, n, np.random.default_rng(seed), 100, 140)
            self.args = (torch.from_numpy(codes).cuda(), torch.from_numpy(tiles).cuda())
            self.values = ops.mxfp4_dequant(*self.args, rows, n)
        else:
            make = synth.q4k_weights if fmt == "q4k" else synth.q4_0_weights
            self.args = (torch.from_numpy(make(rows, n, seed)).cuda(),)
            self.values = getattr(ops, fmt + "_dequant")(*self.args, rows, n)

    def embed(self, ids, **kw):
        return getattr(self.ops, self.fmt + "_embed")(*self.args, ids, self.rows, self.n, **kw)


FORMATS = [("q4k", 1), ("q4k", 5), ("q4_0", 1), ("q4_0", 9), ("q4_0", 127), ("mxfp4", 1), ("mxfp4", 3), ("mxfp4", 130)]


def test_c_entries_refuse_before_any_launch(ffi):
    L, bad = ffi.lib(), ffi.AXC_ERR_INVALID_ARGUMENT
    f32, i32, i64 = ffi.AXC_TY_F32, ffi.AXC_TY_I32, ffi.AXC_TY_I64
    for fn in (L.axc_cuda_q4k_embed, L.axc_cuda_q4_0_embed):
        assert fn(16, 32, f32, 1, 48, f32, 1, 1, 1.0, None, None) == bad          # ids are numbers of 32 or 64 bits
        assert "int32 or int64" in ffi.last_error_detail()
        assert fn(16, 32, i64, 1, 48, i64, 1, 1, 1.0, None, None) == bad
        assert fn(16, 36, i64, 1, 48, f32, 1, 1, 1.0, None, None) == bad          # ids aligned to their type
        assert fn(16, None, i32, 1, 48, f32, 1, 1, 1.0, None, None) == bad
        assert fn(18, 32, i32, 1, 48, f32, 1, 1, 1.0, None, None) == bad
        assert fn(16, 32, i32, 1, 56, f32, 1, 1, 1.0, None, None) == bad
        assert fn(16, 32, i32, 1, 48, f32, 1, 1 << 26, 1.0, None, None) == bad
        assert fn(None, None, i32, 0, None, f32, 1, 1, 1.0, None, None) == ffi.AXC_OK
    assert L.axc_cuda_mxfp4_embed(16, None, 32, i32, 1, 48, f32, 1, 1, 1.0, None, None) == bad
    assert L.axc_cuda_mxfp4_embed(None, None, None, i32, 0, None, f32, 1, 1, 1.0, None, None) == ffi.AXC_OK


def test_python_entries_refuse_cpu_tensors(ops):
    with pytest.raises(ValueError, match="CUDA"):
        ops.q4k_embed(torch.zeros(144, dtype=torch.uint8), torch.zeros(1, dtype=torch.int64), 1, 1)


@gpu
def test_python_entries_refuse_what_does_not_fit(ops, synth):
    q = torch.from_numpy(synth.q4k_weights(4, 1, 1)).cuda()
    ids = torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="q has"):
        ops.q4k_embed(q, ids, 5, 1)
    with pytest.raises(ValueError, match="int32 or int64"):
        ops.q4k_embed(q, ids.to(torch.int16), 4, 1)
    with pytest.raises(ValueError, match="int32 or int64"):
        ops.q4k_embed(q, torch.zeros(4, dtype=torch.int64, device="cuda")[::2], 4, 1)
    with pytest.raises(ValueError, match="int32 or int64"):
        ops.q4k_embed(q, ids.cpu(), 4, 1)
    with pytest.raises(ValueError, match="out has"):
        ops.q4k_embed(q, ids, 4, 1, out=torch.empty(511, device="cuda"))
    with pytest.raises(ValueError, match="out must"):
        ops.q4k_embed(q, ids, 4, 1, out=torch.empty(512, device="cuda"), out_dtype=torch.bfloat16)


@gpu
@pytest.mark.parametrize("fmt,n", FORMATS)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
def test_rows_have_the_bits_of_the_dequantised_table(ops, synth, fmt, n, out_dtype, id_type):
    t = Table(ops, synth, fmt, 200, n, 40 + n)
    ids = torch.randint(0, 200, (77,), device="cuda").to(id_type)
    ids[:4] = torch.tensor([0, 199, 7, 7], device="cuda")
    for scale in (1.0, 0.37, 64.0):
        st = ops.new_status()
        got = t.embed(ids, scale=scale, out_dtype=out_dtype, status=st)
        assert got.shape == (77, t.values.shape[1]) and got.dtype == out_dtype and int(st.item()) == 0
        assert torch.equal(got, (t.values[ids.long()] * scale).to(out_dtype))


@gpu
@pytest.mark.parametrize("fmt,n", [("q4k", 2), ("q4_0", 3), ("mxfp4", 5)])
def test_ids_out_of_range_give_zero_rows_and_a_status_bit(ops, synth, fmt, n):
    t = Table(ops, synth, fmt, 50, n, 60)
    ids = torch.tensor([3, -1, 49, 50, -2 ** 31, 2 ** 31 - 1, 0], device="cuda")
    big = torch.tensor([2 ** 40 + 3, -2 ** 63, 2 ** 63 - 1, 5], dtype=torch.int64, device="cuda")
    for i in (ids.to(torch.int32), ids, big):
        st = ops.new_status()
        out = torch.full((len(i), t.values.shape[1]), 9.0, device="cuda")
        t.embed(i, status=st, out=out)
        fits = (i.long() >= 0) & (i.long() < 50)
        assert int(st.item()) == 2
        assert torch.equal(out[fits], t.values[i.long()[fits]]) and bool((out[~fits] == 0).all())
        t.embed(i)                                        # and without a status word
    assert bool((t.embed(torch.tensor([1], device="cuda"), scale=float("nan"))).isnan().all())


@gpu
def test_shapes_of_ids_and_empty_calls(ops, synth):
    t = Table(ops, synth, "q4k", 10, 1, 61)
    ids = torch.randint(0, 10, (2, 3, 4), device="cuda")
    assert torch.equal(t.embed(ids), t.values[ids])
    assert t.embed(torch.empty(0, dtype=torch.int64, device="cuda")).shape == (0, 256)
    assert t.embed(torch.tensor(4, device="cuda")).shape == (256,)
    out = torch.full((3 * 256 + 64,), 5.0, device="cuda")
    t.embed(ids[0, 0, :3], out=out)
    assert torch.equal(out[:768].view(3, 256), t.values[ids[0, 0, :3]]) and bool((out[768:] == 5.0).all())


@gpu
def test_rows_beyond_four_gigabytes(ops):
    """Byte offsets of rows and outputs that pass 32 bits."""
    rows, n = 70000, 4096                                 # 70000 rows of 65536 bytes of codes: 4.6 GB
    codes = torch.zeros(rows, n * 16, dtype=torch.uint8, device="cuda")
    scales = torch.full((ops.mxfp4_scale_bytes(rows, n),), 127, dtype=torch.uint8, device="cuda")
    for r in (0, 65535, 65536, 69999):
        codes[r] = torch.randint(0, 256, (n * 16,), dtype=torch.uint8, device="cuda")
    ids = torch.tensor([69999, 65536, 65535, 0, 40000], device="cuda")
    got = ops.mxfp4_embed(codes, scales, ids, rows, n, out_dtype=torch.bfloat16)
    point = torch.tensor(list(mx.VALUES), dtype=torch.bfloat16, device="cuda")
    c = codes[ids]
    assert torch.equal(got, point[torch.stack([c & 15, c >> 4], dim=-1).long()].view(5, n * 32))
    many = torch.full((20000,), 3, device="cuda")         # 20000 rows of 262144 bytes out: 5.2 GB
    many[-1], many[16384] = 69999, 65536
    out = ops.mxfp4_embed(codes, scales, many, rows, n, out_dtype=torch.bfloat16)
    assert torch.equal(out[-1], got[0]) and torch.equal(out[16384], got[1]) and bool((out[16385:19999] == 0).all())
    del out
    x = torch.zeros(n * 32, device="cuda")
    x[-1] = 1.0                                           # the last column of every row
    y = ops.mxfp4_matvec(codes, scales, x, rows, n)
    assert torch.equal(y, point[(codes[:, -1] >> 4).long()].float())


@gpu
def test_tied_table_from_embedding_to_head(ops, synth):
    """One MXFP4 table as embedding and as head: rows of the prompt looked up, quantised and multiplied with the table
    again, and the last token's logits by the fp32 matvec; eager, and from a graph with other tokens."""
    rng = np.random.default_rng(70)
    rows, n = 1000, 16
    codes, _s, tiles, w = mx.random_matrix(rows, n, rng)
    c, s = torch.from_numpy(codes).cuda(), torch.from_numpy(tiles).cuda()
    ids = torch.randint(0, rows, (33,), device="cuda")

    def step():
        h = ops.mxfp4_embed(c, s, ids, rows, n, scale=2.0)
        hc, hs = ops.mxfp4_quantize(h)
        return ops.mxfp4_prefill(c, s, hc, hs, 33, rows, n), ops.mxfp4_matvec(c, s, h[-1].contiguous(), rows, n)

    def check(logits, last):
        torch.cuda.synchronize()
        h = 2.0 * w[ids.cpu().numpy()]
        q = mx.values(*mx.quantize(h))
        bound = 2.0 ** -18 * (np.maximum(np.abs(q), np.abs(h)) @ np.abs(w).T)   # 2 x 8 MMA steps of 2^-23 and some sums
        assert (np.abs(logits.double().cpu().numpy() - q @ w.T) <= bound).all()
        assert (np.abs(last.double().cpu().numpy() - h[-1] @ w.T) <= bound[-1] + 2.0 ** -20 * np.abs(h[-1]).max() * np.abs(w).sum(axis=1)).all()

    check(*step())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    ids.copy_(torch.randint(0, rows, (33,), device="cuda"))
    graph.replay()
    check(*out)


@gpu
@pytest.mark.parametrize("fmt,blocks", [("q4k", 2), ("q4_0", 3), ("mxfp4", 5)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_a_table_without_rows_gives_zero_rows(ops, fmt, blocks, out_dtype):
    """Every id is outside it: zeros and the status bit, and nothing is read."""
    e = torch.empty(0, dtype=torch.uint8, device="cuda")
    args = (e, e) if fmt == "mxfp4" else (e,)
    st = ops.new_status()
    cols = blocks * (256 if fmt == "q4k" else 32)
    out = torch.full((3, cols), 9.0, dtype=out_dtype, device="cuda")
    ids = torch.tensor([0, -1, 7], device="cuda")
    getattr(ops, fmt + "_embed")(*args, ids, 0, blocks, out=out, out_dtype=out_dtype, status=st)
    assert bool((out == 0).all()) and int(st.item()) == 2
    assert getattr(ops, fmt + "_embed")(*args, ids[:0], 0, blocks).shape == (0, cols)
