"""The ragged grouped products, 4-bit weights and dropout on the host: the schedule arithmetic and the
generator compiled for the host, the packed layout, and what is refused before anything is launched."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from conftest import ROOT

CSRC = os.path.join(ROOT, "nanospeaker_b200", "csrc")


@pytest.fixture(scope="module")
def lib():
    from nanospeaker_b200 import _lib, build
    build.build()
    return _lib.load()


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """The CUDA-free headers as a host library."""
    d = tmp_path_factory.mktemp("host")
    src = d / "host.cpp"
    src.write_text('''
#include "grouped_order.cuh"
#include "philox.cuh"
extern "C" {
void tile(int l, int m, int n, int band, int* out) {
  const moe::TileAt t = moe::tile_in_bands(l, m, n, band);
  out[0] = t.m; out[1] = t.n;
}
int quotient(int x, int d) { return moe::quotient(x, d, moe::quotient_inverse(d)); }
int chunks(int rows, int ks) { return moe::run_chunks(rows, ks); }
long long chunk_rows(long long rows, int groups, long long tiles, int clusters) {
  return moe::grouped_chunk_rows(rows, groups, tiles, clusters);
}
void philox(unsigned long long low, unsigned long long high, unsigned long long key, unsigned* w) {
  const uint64_t at = low;
  moe::philox4x32<1>(&at, high, key, reinterpret_cast<uint32_t(*)[4]>(w));
}
void philox4(unsigned long long low, unsigned long long high, unsigned long long key, unsigned* w) {
  const uint64_t at[4] = {low, low + 1, low + 2, low + 3};
  moe::philox4x32<4>(at, high, key, reinterpret_cast<uint32_t(*)[4]>(w));
}
unsigned threshold(double p) { return moe::dropout_threshold(p); }
}
''')
    so = d / "host.so"
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-std=c++17", f"-I{CSRC}", str(src), "-o", str(so)],
                   check=True)
    lib = ctypes.CDLL(str(so))
    lib.chunk_rows.restype = ctypes.c_longlong
    lib.chunk_rows.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_longlong, ctypes.c_int]
    lib.philox.argtypes = lib.philox4.argtypes = [ctypes.c_ulonglong] * 3 + [ctypes.c_void_p]
    lib.threshold.restype = ctypes.c_uint
    lib.threshold.argtypes = [ctypes.c_double]
    return lib


# ------------------------------------------------------------------------------------ schedules
@pytest.mark.parametrize("m,n,band", [(1, 1, 8), (8, 3, 8), (9, 5, 8), (128, 16, 8), (3, 64, 8), (7, 1, 4)])
def test_every_tile_is_walked_once_and_bands_stay_together(host, m, n, band):
    at = (ctypes.c_int * 2)()
    seen = []
    for l in range(m * n):
        host.tile(l, m, n, band, at)
        seen.append((at[0], at[1]))
    assert sorted(seen) == [(i, j) for i in range(m) for j in range(n)]
    bands = [i // band for i, _ in seen]
    assert bands == sorted(bands)


def test_quotients(host):
    for d in (1, 2, 3, 5, 7, 12, 96, 127, 1000, 65535, 1 << 20, (1 << 31) - 1):
        for x in [0, 1, d - 1, d, 2 * d - 1, 2 * d, (1 << 31) - 1, (1 << 31) // d * d - 1, (1 << 31) // d * d]:
            if 0 <= x < 1 << 31:
                assert host.quotient(x, d) == x // d


@pytest.mark.parametrize("rows,ks,want", [(0, 512, 1), (1, 512, 1), (512, 512, 1), (513, 512, 2),
                                          (1025, 512, 3)])
def test_chunks_of_a_run(host, rows, ks, want):
    assert host.chunks(rows, ks) == want


def test_chunks_of_the_longest_run(host):
    rows = (1 << 31) - 257
    for ks in (256, 1 << 20, 96_745_344, rows - 1, rows):
        assert host.chunks(rows, ks) == -(-rows // ks)


def test_chunk_rows(host):
    """Runs are cut where there are too few tiles for the clusters, or where one is far longer than the
    rest."""
    ks = lambda rows, groups, tiles: host.chunk_rows(rows, groups, tiles, 74)  # noqa: E731
    for rows, groups, tiles in ((1, 1, 1), (98304, 76, 3), (32768, 16, 128), (1 << 20, 1, 1), (5, 1024, 9)):
        assert ks(rows, groups, tiles) % 64 == 0 and ks(rows, groups, tiles) >= 256
    assert ks(98304, 76, 3) >= 2 * 98304 // 76             # many tiles: only long runs
    assert ks(98304, 76, 3) <= 98304 * 3 // 74             # but those
    assert ks(102400, 8, 2) <= 12800 // 3                  # sixteen tiles, 74 clusters
    assert ks(1 << 20, 1, 1) <= (1 << 20) // 16


def test_scratch_covers_every_split_run(lib, host):
    """Whatever the runs are, the chunks of split runs fit the scratch."""
    rng = torch.Generator().manual_seed(0)
    for rows, m, n, groups in ((98304, 576, 256, 76), (5000, 64, 64, 3), (20000, 8, 8, 1000)):
        tiles = -(-m // 256) * -(-n // (256 if n > 128 else 128))
        ks = host.chunk_rows(rows, groups, tiles, 74)
        each = tiles * 256 * (256 if n > 128 else 128) * 4
        have = lib.moe_b200_grouped_wgrad_scratch_bytes(m, n, rows, groups) // each
        for skew in (0.0, 1.0, 20.0):
            load = torch.softmax(torch.randn(groups, generator=rng) * skew, 0)
            counts = torch.bincount(torch.multinomial(load, rows, True, generator=rng), minlength=groups)
            need = sum(host.chunks(int(c), ks) for c in counts if c > ks)
            assert need <= have


def test_pair_kernels_begin_in_the_one_place():
    """A kernel of CTA pairs lets the next one in when it holds its TMEM and reads nothing before its wait: the
    order stands in pair_start, and the kernels here begin with it and nothing else of it."""
    code = lambda f: re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, f)).read())  # noqa: E731
    body = code("pair.cuh").split("pair_start(")[1].split("\n}\n")[0]
    assert re.findall(r"\b(tmem_alloc|tmem_relinquish|pdl_trigger|cluster_sync_all|pdl_wait)2?\(", body) == [
        "tmem_alloc", "tmem_relinquish", "pdl_trigger", "cluster_sync_all", "pdl_wait"]
    kernels = [k.split("\n}\n")[0] for k in code("grouped.cu").split("__global__")[1:]]
    pairs = [k for k in kernels if "tmem_dealloc2" in k]
    assert len(pairs) == 2
    for k in pairs:
        assert k.count("pair_start(") == 1 and not re.search(r"tmem_alloc|pdl_trigger|pdl_wait", k)
        assert "p.offsets" not in k.split("pair_start(")[0]


# ------------------------------------------------------------------------------------ generator
# The published known answers of Philox4x32-10 (counter words, key words, output words).
PHILOX_ANSWERS = [
    ([0, 0, 0, 0], [0, 0], [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
    ([0xffffffff] * 4, [0xffffffff] * 2, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
    ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0],
     [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]),
]


@pytest.mark.parametrize("counter,key,want", PHILOX_ANSWERS)
def test_philox_known_answers(host, counter, key, want):
    w = (ctypes.c_uint * 4)()
    host.philox(counter[0] | counter[1] << 32, counter[2] | counter[3] << 32, key[0] | key[1] << 32, w)
    assert list(w) == want


def test_counters_side_by_side_are_the_single_ones(host):
    for low in (0, 12, (1 << 32) - 4, 1 << 32, 0x123456789ABCDEF0):
        four, one = (ctypes.c_uint * 16)(), (ctypes.c_uint * 4)()
        host.philox4(low, 77, 0x1122334455667788, four)
        for j in range(4):
            host.philox(low + j, 77, 0x1122334455667788, one)
            assert list(four[4 * j:4 * j + 4]) == list(one)


def test_thresholds(host):
    for p in (0.0, 0.1, 0.25, 0.5, 1 / 3, 0.9, 2.0 ** -33, 3 * 2.0 ** -33, 1 - 2.0 ** -40):
        assert host.threshold(p) == min(round(p * 2 ** 32), 2 ** 32 - 1)


# --------------------------------------------------------------------------------- 4-bit weights
@pytest.mark.parametrize("shape,group", [((8, 1), 32), ((64, 16), 64), ((1000, 1537), 32), ((576, 256), 64),
                                         ((3, 128, 40), 64), ((2, 72, 16), 128), ((1, 200, 33), 128)])
def test_packing_returns_what_was_packed(shape, group):
    from nanospeaker_b200 import Int4Weight
    levels = torch.randint(0, 16, shape, dtype=torch.uint8)
    k, n = shape[-2:]
    scales = torch.rand(*shape[:-2], -(-k // group), n).bfloat16()
    w = Int4Weight.from_levels(levels, scales, group)
    back, s = w.to_levels()
    assert torch.equal(back, levels) and torch.equal(s, scales)
    assert w.data.dtype == torch.uint8 and w.data.is_contiguous()
    assert w.shape == shape and w.dtype == torch.bfloat16


@pytest.mark.parametrize("k,group", [(128, 64), (576, 128), (640, 32), (1024, 64)])
def test_packed_layout_is_the_documented_one(lib, k, group):
    """Chunk by chunk, strip by strip: nibble i of half b of word j of lane 4 * row + t, then the scales."""
    from nanospeaker_b200 import Int4Weight
    levels = torch.randint(0, 16, (k, 32), dtype=torch.uint8)
    scales = torch.rand(-(-k // group), 32).half()
    w = Int4Weight.from_levels(levels, scales, group)
    data = bytes(w.data[0].tolist())
    assert len(data) == lib.moe_b200_int4_bytes(k, 32, group)
    at, kb = 0, k // 64
    for chunk in range(0, kb, 8):
        blocks = range(chunk, min(kb, chunk + 8))
        groups = range(chunk * 64 // group, -(-blocks.stop * 64 // group))
        for strip in range(2):
            for block in blocks:
                for lane in range(32):
                    row, t = lane // 4, lane % 4
                    for j in range(4):
                        word = int.from_bytes(data[at:at + 4], "little")
                        at += 4
                        for i in range(4):
                            for b in range(2):
                                into = 64 * block + 32 * (j // 2) + 8 * t + 4 * (j % 2) + 2 * (i // 2) + b
                                assert (word >> (4 * i + 16 * b)) & 15 == \
                                    int(levels[into, 16 * strip + row + 8 * (i % 2)])
            for g in groups:
                for row in range(8):
                    for i in range(2):
                        v = torch.frombuffer(bytearray(data[at:at + 2]), dtype=torch.float16)
                        at += 2
                        assert v == scales[g, 16 * strip + row + 8 * i]
    assert at == len(data)


def test_packed_bytes(lib):
    assert lib.moe_b200_int4_bytes(4096, 4096, 128) == 4096 * 4096 // 2 + 4096 * 32 * 2
    for k, n, group in ((60, 16, 64), (64, 0, 64), (64, 16, 96), (0, 16, 32)):
        assert lib.moe_b200_int4_bytes(k, n, group) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantisation_is_within_half_a_level(dtype, group):
    """scale = largest / 7 rounded to 16 bits (relative 2^-8 at most): a level is at most half a scale
    off, and the largest value, at 7 scales, at most 7 * 2^-8 of a scale more."""
    from nanospeaker_b200 import quantize_int4
    w = (torch.randn(2, 200, 48) * 0.1).to(dtype)
    q = quantize_int4(w, group)
    assert q.dtype == (torch.bfloat16 if dtype == torch.float32 else dtype)
    _, scales = q.to_levels()
    each = scales.float().repeat_interleave(group, 1)[:, :200]
    assert ((q.dequantize() - w.float()).abs() <= each * (0.5 + 7 * 2.0 ** -8) * (1 + 1e-6)).all()


def test_quantising_zeros_and_what_is_not_finite():
    from nanospeaker_b200 import quantize_int4
    assert (quantize_int4(torch.zeros(64, 16)).dequantize() == 0).all()
    for bad in (float("inf"), float("nan")):
        w = torch.zeros(64, 16)
        w[3, 5] = bad
        with pytest.raises(ValueError, match="infinities or NaN"):
            quantize_int4(w)


def test_scales_that_overflow_are_refused():
    from nanospeaker_b200 import quantize_int4
    w = torch.full((64, 16), 1e6)
    with pytest.raises(ValueError, match="too large"):
        quantize_int4(w, 64, torch.float16)
    assert torch.allclose(quantize_int4(w, 64, torch.bfloat16).dequantize(), w, rtol=2.0 ** -7)


def test_weight_refusals():
    from nanospeaker_b200 import Int4Weight, quantize_int4
    q, s = torch.zeros(64, 16, dtype=torch.uint8), torch.ones(1, 16).half()
    for group in (0, 16, 33, 96, 256):
        with pytest.raises(ValueError, match="scale groups"):
            Int4Weight.from_levels(q, s, group)
    with pytest.raises(ValueError, match="uint8"):
        Int4Weight.from_levels(q.int(), s, 64)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        Int4Weight.from_levels(q, s.float(), 64)
    with pytest.raises(ValueError, match="do not take scales"):
        Int4Weight.from_levels(q, s, 32)
    with pytest.raises(ValueError, match="multiple of 8"):
        quantize_int4(torch.randn(60, 16))
    with pytest.raises(ValueError, match=r"\[K, N\]"):
        quantize_int4(torch.randn(60))


# ------------------------------------------------------------------------------------- refusals
def test_packed_weights_that_are_not_what_they_say_are_refused(lib):
    from nanospeaker_b200 import Int4Weight, quantize_int4
    from nanospeaker_b200.int4 import _matrix_bytes
    for k, n, group in ((8, 1, 32), (136, 33, 128), (4096, 4096, 64), (520, 17, 128), (1000, 16, 32)):
        assert _matrix_bytes(k, n, group) == lib.moe_b200_int4_bytes(k, n, group)
    w = quantize_int4(torch.randn(3, 128, 48), 64)
    again = Int4Weight(w.data, w.shape, w.group, w.dtype)
    assert torch.equal(again.dequantize(), w.dequantize())
    for data, shape, group, dtype, what in (
            (w.data[:2], w.shape, 64, w.dtype, "in one piece"),
            (w.data[:, :-32], w.shape, 64, w.dtype, "in one piece"),
            (w.data, (3, 128, 64), 64, w.dtype, "in one piece"),
            (w.data, w.shape, 32, w.dtype, "in one piece"),
            (w.data.to(torch.int32), w.shape, 64, w.dtype, "in one piece"),
            (w.data.t().contiguous().t(), w.shape, 64, w.dtype, "in one piece"),
            (w.data, w.shape, 48, w.dtype, "scale groups"),
            (w.data, w.shape, 64, torch.float32, "scales are"),
            (w.data, (384, 3, 16, 8), 64, w.dtype, "a weight is"),
            (w.data, (3, 130, 48), 64, w.dtype, "multiple of 8")):
        with pytest.raises(ValueError, match=what):
            Int4Weight(data, shape, group, dtype)
    off = torch.empty(w.data.numel() + 1, dtype=torch.uint8)[1:].view(w.data.shape)
    with pytest.raises(ValueError, match="16 bytes"):
        Int4Weight(off, w.shape, 64, w.dtype)
    with pytest.raises(ValueError, match="0 .. 15"):
        Int4Weight.from_levels(torch.full((64, 16), 16, dtype=torch.uint8), torch.ones(1, 16, dtype=torch.bfloat16), 64)


def test_grouped_refusals():
    from nanospeaker_b200 import grouped_mm
    x, w = torch.randn(6, 16).bfloat16(), torch.randn(2, 16, 24).bfloat16()
    off = torch.tensor([0, 2, 6], dtype=torch.int32)
    bad = lambda msg, *a: _refused(grouped_mm, msg, *a)  # noqa: E731
    bad("takes x", x[0], w, off)
    bad("takes x", x, w[0], off)
    bad("fit together", x, w, off[:2])
    bad("fit together", x[:, :8], w, off)
    bad("bf16 or fp16", x.float(), w.float(), off)
    bad("bf16 or fp16", x, w.half(), off)
    bad("int32", x, w, off.long())
    bad("multiples of 8", x, w[:, :, :20], off)
    bad("multiples of 8", torch.randn(6, 12).bfloat16(), torch.randn(2, 12, 16).bfloat16(), off)
    bad("groups", torch.randn(1, 8).half(), torch.randn(1025, 8, 8).half(),
        torch.zeros(1026, dtype=torch.int32))
    bad("CUDA device", x, w, off)


def _refused(fn, msg, *a, **kw):
    with pytest.raises(ValueError, match=msg):
        fn(*a, **kw)


def test_int4_refusals():
    from nanospeaker_b200 import int4_experts, int4_mm, quantize_int4
    x = torch.randn(3, 64).half()
    w = quantize_int4(torch.randn(64, 32).half())
    with pytest.raises(TypeError):
        int4_experts(x, x[:, :1], torch.zeros(3, 1, dtype=torch.int64), w, torch.zeros(3))
    _refused(int4_mm, "one matrix", x, quantize_int4(torch.randn(2, 64, 32).half()))
    _refused(int4_mm, "one matrix", x[:, :32], w)
    _refused(int4_mm, "have to be alike", x.bfloat16(), w)
    _refused(int4_mm, "CUDA device", x, w)
    w_in, w_out = quantize_int4(torch.randn(4, 64, 64).half()), quantize_int4(torch.randn(4, 32, 64).half())
    tw, idx = torch.ones(3, 2).half(), torch.zeros(3, 2, dtype=torch.int64)
    _refused(int4_experts, "no kernel", x, tw, idx, w_in, w_out, activation="cube")
    _refused(int4_experts, "takes x", x, tw, idx[:2], w_in, w_out)
    _refused(int4_experts, "int64", x, tw, idx.int(), w_in, w_out)
    _refused(int4_experts, "int64", x, tw.float(), idx, w_in, w_out)
    _refused(int4_experts, "do not fit", x, tw, idx, w_out, w_in)
    _refused(int4_experts, "do not fit", x[:, :32].contiguous(), tw, idx, w_in, w_out)
    _refused(int4_experts, "do not fit", x, tw, idx, w_in, w_out, shared_in=w_out, shared_out=w_out)
    _refused(int4_experts, "multiple of 16", x, tw, idx, quantize_int4(torch.randn(4, 64, 48).half()),
             quantize_int4(torch.randn(4, 24, 64).half()))
    _refused(int4_experts, "different sizes", x, tw, idx, w_in, quantize_int4(torch.randn(4, 32, 64).half(), 32))
    _refused(int4_experts, "CUDA device", x, tw, idx, w_in, w_out)
    with pytest.raises(TypeError):
        int4_experts(x, tw, idx, w_in, w_out, shared_in=w_in)


def test_dropout_refusals():
    from nanospeaker_b200 import dropout_add
    x, rng = torch.randn(4, 4), torch.zeros(2, dtype=torch.int64)
    _refused(dropout_add, "fp32", x.double(), None, 0.1, rng)
    _refused(dropout_add, "residual", x, x[:2], 0.1, rng)
    _refused(dropout_add, "residual", x, x.half(), 0.1, rng)
    for p in (-0.1, 1.0, 1.5, float("nan")):
        _refused(dropout_add, "has to be in", x, None, p, rng)
    _refused(dropout_add, "int64", x, None, 0.1, rng.int())
    _refused(dropout_add, "int64", x, None, 0.1, torch.zeros(3, dtype=torch.int64))
    _refused(dropout_add, "CUDA device", x, None, 0.1, rng)


def test_entry_points_validate_before_any_launch(lib):
    """Bad shapes, types, pointers and scratch come back as error codes (no GPU needed)."""
    buf = ctypes.create_string_buffer(256)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 63) & ~63)
    odd = ctypes.c_void_p(p.value + 2)
    null = ctypes.c_void_p(0)
    mm = lambda x=p, rows=4, ld=64, k=64, w=p, g=2, gs=64 * 32, ldw=32, n=32, off=p, dt=0, y=p, st=p: \
        lib.moe_b200_grouped_mm(x, rows, ld, k, w, g, gs, ldw, 1, n, off, dt, y, st, null)  # noqa: E731
    assert mm(rows=0) == 0
    assert mm(rows=-1) == mm(k=60) == mm(n=30) == mm(g=0) == mm(g=1025) == mm(ld=63) == mm(ld=56) == -1
    assert mm(ldw=24) == mm(gs=33) == mm(rows=1 << 31) == -1
    assert mm(dt=2) == mm(dt=-1) == -5
    assert mm(x=null) == mm(w=null) == mm(off=null) == mm(y=null) == mm(st=null) == -2
    assert mm(x=odd) == mm(w=odd) == mm(y=odd) == mm(off=odd) == -3
    wg = lambda a=p, lda=64, m=64, b=p, ldb=32, n=32, rows=4, off=p, g=2, dt=0, dw=p, sc=null, nb=0, st=p: \
        lib.moe_b200_grouped_wgrad(a, lda, m, b, ldb, n, rows, off, g, dt, dw, sc, nb, st, null)  # noqa: E731
    assert wg(rows=-1) == wg(m=60) == wg(n=4) == wg(g=0) == wg(lda=56) == wg(ldb=28) == -1
    assert wg(dt=2) == -5
    assert wg(a=null) == wg(b=null) == wg(off=null) == wg(dw=null) == wg(st=null) == -2
    assert wg(a=odd) == wg(b=odd) == wg(dw=odd) == -3
    need = lib.moe_b200_grouped_wgrad_scratch_bytes(64, 32, 100000, 2)
    assert need > 0 and lib.moe_b200_grouped_wgrad_scratch_bytes(64, 32, 256, 2) == 0
    assert wg(rows=100000) == wg(rows=100000, sc=p, nb=need - 1) == -4
    q = lambda x=p, rows=4, ld=64, k=64, w=p, grp=64, n=32, dt=0, y=p, st=p: \
        lib.moe_b200_int4_mm(x, rows, ld, k, w, grp, n, dt, y, st, null)  # noqa: E731
    assert q(rows=0) == 0
    assert q(rows=-1) == q(k=60) == q(n=0) == q(ld=56) == q(grp=16) == q(grp=96) == q(grp=256) == -1
    assert q(dt=2) == -5
    assert q(x=null) == q(w=null) == q(y=null) == q(st=null) == -2
    assert q(x=odd) == q(w=odd) == -3
    ex = lambda t=4, d=64, h=32, k=2, e=4, s=0, w=p, idx=p, grp=64, act=0, dt=0, sc=p, nb=1 << 20, sh=null, o=p: \
        lib.moe_b200_int4_experts(p, t, d, d, h, w, idx, k, e, p, p, s, sh, sh, grp, act,
                                  dt, o, sc, nb, p, null)  # noqa: E731
    assert ex(t=0) == 0
    assert ex(t=-1) == ex(d=60) == ex(h=24) == ex(k=0) == ex(e=0) == ex(s=-1) == ex(grp=48) == -1
    assert ex(e=65536) == ex(t=1 << 30) == -1
    assert ex(dt=2) == ex(act=5) == ex(act=-1) == -5
    assert ex(w=null) == ex(idx=null) == ex(o=null) == ex(s=1) == -2
    assert ex(o=odd) == ex(idx=odd) == -3
    bytes_ = lib.moe_b200_int4_experts_scratch_bytes(4, 2, 1, 64, 32)
    assert bytes_ >= 12 * (32 * 2 + 64 * 4)
    assert ex(s=1, sh=p, nb=bytes_ - 1) == ex(sc=null) == -4
    dr = lambda x=p, r=null, n=8, dt=0, pr=0.1, rng=p, used=null, o=p: \
        lib.moe_b200_dropout(x, r, n, dt, pr, rng, used, o, null)  # noqa: E731
    assert dr(n=0) == 0
    assert dr(n=-1) == dr(pr=1.0) == dr(pr=-0.5) == dr(pr=float("nan")) == -1
    assert dr(dt=3) == -5
    assert dr(x=null) == dr(rng=null) == dr(o=null) == -2
    assert dr(rng=odd) == dr(used=odd) == dr(x=odd, dt=2) == -3


def test_sizes_whose_places_leave_31_bits_are_refused(lib):
    buf = ctypes.create_string_buffer(256)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 63) & ~63)
    rows = (1 << 31) - 256
    assert lib.moe_b200_grouped_mm(p, rows, 8, 8, p, 1, 64, 8, 1, 8, p, 0, p, p, None) == -1
    assert lib.moe_b200_grouped_wgrad(p, 8, 8, p, 8, 8, rows, p, 1, 0, p, None, 0, p, None) == -1
    for tokens, top_k in (((1 << 31) - 1023, 1), (1, (1 << 31) - 1023), ((1 << 33) + 1, 1)):
        assert lib.moe_b200_int4_experts(p, tokens, 8, 8, 16, p, p, top_k, 4, p, p, 0, None, None, 64, 0, 0, p, p,
                                         1 << 62, p, None) == -1
    for many in (65535 * 32 + 1, (1 << 31) - 1):
        assert lib.moe_b200_int4_mm(p, many, 8, 8, p, 64, 8, 0, p, p, None) == -5
    from nanospeaker_b200 import grouped_mm
    x, w = torch.empty(4, 1 << 31, device="meta", dtype=torch.bfloat16), torch.empty(
        2, 1 << 31, 8, device="meta", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="widths"):
        grouped_mm(x, w, torch.empty(3, device="meta", dtype=torch.int32))


def test_products_of_more_tiles_than_31_bits_count_are_refused(lib):
    """One row and two widths of 2^24, nothing to split: 2^32 tiles, which 32 bits take for none."""
    buf = ctypes.create_string_buffer(256)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 63) & ~63)
    for m, n, groups in ((1 << 24, 1 << 24, 1), (1 << 30, 1 << 30, 1024), (1 << 19, 1 << 19, 1024)):
        assert lib.moe_b200_grouped_wgrad(p, m, m, p, n, n, 1, p, groups, 0, p, None, 0, p, None) == -5
        assert lib.moe_b200_grouped_wgrad(p, m, m, p, n, n, (1 << 31) - 257, p, groups, 0, p, None, 1 << 62, p,
                                          None) in (-4, -5)
    assert lib.moe_b200_grouped_wgrad_scratch_bytes(1 << 24, 1 << 24, 1 << 30, 1) == 0


def test_widths_whose_last_tile_leaves_31_bits_are_refused(lib):
    """Widths just below 2^31: what is rounded up to whole tiles or strips would be negative."""
    buf = ctypes.create_string_buffer(256)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 63) & ~63)
    wide = (1 << 31) - 8
    mm = lambda k, n: lib.moe_b200_grouped_mm(p, 1, k, k, p, 1, k * n, n, 1, n, p, 0, p, p, None)  # noqa: E731
    wg = lambda m, n: lib.moe_b200_grouped_wgrad(p, m, m, p, n, n, 1, p, 1, 0, p, None, 0, p, None)  # noqa: E731
    assert mm(wide, 8) == mm(8, wide) == wg(wide, 8) == wg(8, wide) == -1
    assert lib.moe_b200_grouped_wgrad_scratch_bytes(wide, 8, 1 << 20, 1) == 0
    odd = (1 << 31) - 1
    q = lambda k, n: lib.moe_b200_int4_mm(p, 1, k, k, p, 64, n, 0, p, p, None)  # noqa: E731
    assert q(wide, 8) == q(8, odd) == -1
    assert lib.moe_b200_int4_bytes(wide, 8, 64) == lib.moe_b200_int4_bytes(8, odd, 64) == 0
    assert lib.moe_b200_int4_bytes(8, (1 << 31) - 257, 128) == (((1 << 31) - 257 + 15) // 16) * (512 + 32)
    for d, h in ((wide, 16), (64, 1 << 30), (64, (1 << 31) - 16)):
        assert lib.moe_b200_int4_experts(p, 1, d, d, h, p, p, 1, 4, p, p, 0, None, None, 64, 0, 0, p, p, 1 << 62, p,
                                         None) == -1
    from nanospeaker_b200 import Int4Weight, grouped_mm
    meta = lambda *s: torch.empty(*s, device="meta", dtype=torch.bfloat16)  # noqa: E731
    off = torch.empty(2, device="meta", dtype=torch.int32)
    _refused(grouped_mm, "widths", meta(1, wide), meta(1, wide, 8), off)
    _refused(grouped_mm, "widths", meta(1, 8), meta(1, 8, wide), off)
    _refused(Int4Weight, "outputs", torch.empty(1, 64, device="meta", dtype=torch.uint8), (8, odd), 64, torch.bfloat16)


def test_status_word_of_a_call_in_inference_mode():
    """A word that a serving call makes first is read and set back outside inference mode as well."""
    from nanospeaker_b200 import kernels
    dev = torch.device("cpu", 7)
    with torch.inference_mode():
        word = kernels.status_word(dev)
    word.fill_(2)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="expert id"):
            kernels.check_status(dev)
        kernels.check_status(dev)
        with torch.inference_mode():
            kernels.status_word(dev).fill_(2)
    kernels._status_words.pop(("cpu", 7))


def low_level_calls(device):
    """Every low-level entry, by its function or its registered op, with one operand that does not have the length
    that another gives it."""
    from nanospeaker_b200 import kernels as K
    from nanospeaker_b200 import quantize_int4
    half = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=device)  # noqa: E731
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=device)  # noqa: E731
    x, w, idx = half(6, 64), half(2, 64, 24), torch.zeros(6, 2, dtype=torch.int64, device=device)
    one = quantize_int4(torch.zeros(64, 32)).data.to(device)
    w_in = quantize_int4(torch.zeros(4, 64, 64)).data.to(device)
    w_out = quantize_int4(torch.zeros(4, 32, 64)).data.to(device)
    sh_in, sh_out = w_in[:1], w_out[:1]
    rng = torch.zeros(2, dtype=torch.int64, device=device)
    ops = torch.ops.moe_b200
    for mm in (K.grouped_mm, ops.grouped_mm):
        yield from ((mm, a) for a in ((half(1, 32), w, i32(3)), (x, w, i32(2)), (x, w, i32(3).long()),
                                      (x, w.half(), i32(3)), (x[0], w, i32(3))))
    yield K.grouped_mm, (x, w, i32(6)[::2])
    yield K.grouped_mm, (x, w.to("meta"), i32(3))
    for wg in (K.grouped_wgrad, ops.grouped_wgrad):
        yield from ((wg, a) for a in ((x, half(5, 24), i32(3)), (x, half(7, 24), i32(3)), (x, half(6, 24).half(), i32(3)),
                                      (x, half(6, 24), i32(3).long()), (x, half(6, 24), i32(1))))
    for mm in (K.int4_mm, ops.int4_mm):
        yield from ((mm, a) for a in ((x, one, 64, 48), (x, one, 32, 32), (half(6, 128), one, 64, 32), (x, one, 48, 32),
                                      (x, one[:, :-32], 64, 32), (x, one.view(torch.int8), 64, 32),
                                      (x[0], one, 64, 32)))
    for ex in (K.int4_experts, ops.int4_experts):
        good = [x, half(6, 2), idx, w_in, w_out, sh_in, sh_out, 32, 64, 0]
        for at, other in ((0, half(5, 64)), (0, half(6, 128)), (1, half(6, 1)), (1, half(6, 2).half()), (2, idx.int()),
                          (3, w_in[:3]), (4, w_out[:3]), (5, None), (6, None), (5, w_in[:2]), (7, 48), (8, 32)):
            yield ex, (*good[:at], other, *good[at + 1:])
    yield from ((K.dropout, a) for a in ((x, half(6, 32), 0.1, rng), (x, x.half(), 0.1, rng), (x, None, 0.1, rng[:1]),
                                         (x, None, 0.1, rng.int()), (x, None, 0.1, rng, rng[:1])))
    yield ops.dropout_add, (x, half(6, 32), 0.1, rng)
    yield ops.dropout_bwd, (x, 0.1, rng[:1])


def test_low_level_entries_refuse_operands_that_do_not_fit():
    """Before the device is looked at: what they would read past the end of is never reached."""
    n = 0
    for call, args in low_level_calls("cpu"):
        if not isinstance(call, torch._ops.OpOverloadPacket):     # (the ops take CUDA tensors alone)
            with pytest.raises(ValueError, match="do not fit together"):
                call(*args)
            n += 1
    assert n > 30


@pytest.mark.parametrize("how", ["dual", "jvp"])
def test_forward_mode_is_refused(how):
    """An operand with a tangent requires no gradient as a rule; its tangent would be dropped without a word."""
    import torch.autograd.forward_ad as fwad
    from nanospeaker_b200 import dropout_add, fused_moe_forward, grouped_mm, int4_experts, int4_mm, quantize_int4
    half = lambda *s: torch.randn(*s).bfloat16()  # noqa: E731
    w, off, one = half(2, 16, 24), torch.tensor([0, 2, 6], dtype=torch.int32), quantize_int4(half(16, 8))
    w_in, w_out = quantize_int4(half(2, 16, 32)), quantize_int4(half(2, 16, 16))
    tw, idx, rng = half(6, 1), torch.zeros(6, 1, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)
    x = half(6, 16)
    calls = ((lambda v: grouped_mm(v, w, off), x), (lambda v: grouped_mm(x, v, off), w), (lambda v: int4_mm(v, one), x),
             (lambda v: int4_experts(v, tw, idx, w_in, w_out), x), (lambda v: int4_experts(x, v, idx, w_in, w_out), tw),
             (lambda v: dropout_add(v, None, 0.1, rng), x), (lambda v: dropout_add(x, v, 0.1, rng), x),
             (lambda v: fused_moe_forward(v, half(2, 16, 32), half(2, 16, 16), tw, idx, None, None, "silu"), x))
    for call, at in calls:
        with pytest.raises(NotImplementedError, match="forward mode"):
            if how == "jvp":
                torch.func.jvp(call, (at,), (torch.ones_like(at),))
            else:
                with fwad.dual_level():
                    call(fwad.make_dual(at, torch.ones_like(at)))
