"""Products of 4-bit matrices, norms and gates with 8-bit rows, against float64."""

import numpy as np
import pytest
import torch

import plain_mx

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def mx():
    from liyab_amd.kernels import mx as module

    return module


def rnd(*shape, seed=0, scale=1.0, dtype=torch.float32):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


def matrix(mx, N, K, seed=0, scale=0.1):
    """(the matrix, its values in float64): from plain rows made by the plain implementation, a group in eight far smaller than the others."""
    rng = np.random.default_rng(seed)
    w = rng.normal(size=(N, K)) * scale * np.exp2(rng.integers(-8, 1, size=(N, 1)) * (rng.random((N, 1)) < 0.125))
    codes, scales = plain_mx.quantize(w, plain_mx.E2M1, 2)
    m = mx.Mxfp4Matrix.pack(torch.from_numpy(plain_mx.two_a_byte(codes)).to(DEV), torch.from_numpy(scales).to(DEV), K)
    return m, plain_mx.values(codes, scales, plain_mx.E2M1)


def rows_of(mx, M, K, kind, seed=1):
    """(what the product takes, its values in float64)."""
    if kind == "mxfp8":
        codes, scales = plain_mx.quantize(np.random.default_rng(seed).normal(size=(M, K)), plain_mx.E4M3, 8)
        return mx.Mxfp8Rows.pack(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV)), plain_mx.values(codes, scales, plain_mx.E4M3)
    a = rnd(M, K, seed=seed, dtype=getattr(torch, kind))
    return a, a.double().cpu().numpy()


def within(got, want, bound, what):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all(), what
    off = np.abs(got - want) / bound
    assert off.max() <= 1, f"{what}: {off.max():.3g} of the bound at {np.unravel_index(off.argmax(), off.shape)}"


def sums_bound(a, w, bias, K, cut=False):
    """Products are exact in 32 bits; every partial sum is off by at most a unit in the last place of what it can reach, in at most K / 4 + 64 steps (4 k an instruction in
    float32, the waves' sums and the bias behind them). `cut`: the scaled matrix instruction (8-bit rows, more than 64 of them) adds eight neighbouring products without what lies
    below 2^-13 of the largest: each is off by less than that, eight of them by 2^-10 of the largest, which their sizes' sum is no less than."""
    return (2.0 ** -10 * cut + (K / 4 + 64) * 2.0 ** -23) * (np.abs(a) @ np.abs(w).T + np.abs(bias)) + 1e-30


HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}

# one of everything; a strip's, a tile's and a chunk's edges, K of no whole chunk, group or piece, the sizes at which another number of rows a workgroup is taken
SHAPES = [(1, 1, 1), (1, 16, 128), (2, 17, 40), (5, 100, 129), (15, 33, 256), (16, 64, 1600), (17, 48, 97), (31, 80, 512), (33, 40, 640), (64, 130, 2080), (65, 96, 1000),
          (100, 257, 384), (130, 300, 576), (257, 272, 264)]


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "mxfp8"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_products(mx, M, N, K, kind):
    w, wv = matrix(mx, N, K)
    a, av = rows_of(mx, M, K, kind)
    bias = rnd(N, seed=2)
    b = bias.double().cpu().numpy()
    cut = kind == "mxfp8" and M > 64
    want, bound = av @ wv.T + b, sums_bound(av, wv, b, K, cut)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((M, N), float("nan"), dtype=dtype, device=DEV)
        mx.gemm_mx(a, w, bias, out=out)
        within(out, want, bound + HALF[dtype] * (np.abs(want) + bound), f"{kind} -> {dtype}")
    out = torch.full((M, N + 8), 3.0, device=DEV)
    mx.gemm_mx(a, w, None, out=out[:, 4:N + 4])  # rows of a wider buffer; nothing beside them
    within(out[:, 4:N + 4], av @ wv.T, bound + HALF[torch.float32] * (np.abs(want) + np.abs(b)), "no bias")
    assert (out[:, :4] == 3).all() and (out[:, N + 4:] == 3).all()
    stream = rnd(M, N, seed=3)
    before = stream.double().cpu().numpy()
    mx.gemm_mx(a, w, bias, residual=stream)
    within(stream, before + want, bound + HALF[torch.float32] * (np.abs(before) + np.abs(want) + bound), "residual")


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "mxfp8"])
@pytest.mark.parametrize("activation", ["gelu_tanh", "gelu_erf"])
@pytest.mark.parametrize("M,N,K", [(3, 70, 96), (40, 50, 256), (150, 260, 320)])
def test_activations(mx, M, N, K, activation, kind):
    """The activation's slope is below 1.13; its own 32-bit evaluation: 2^-18 of the argument, whose exponential takes arguments up to 2^7 with their rounding."""
    w, wv = matrix(mx, N, K, scale=0.3)
    a, av = rows_of(mx, M, K, kind)
    bias = rnd(N, seed=2)
    b = bias.double().cpu().numpy()
    v = av @ wv.T + b
    want, bound = plain_mx.gelu(v, activation), 1.13 * sums_bound(av, wv, b, K, kind == "mxfp8" and M > 64) + 2.0 ** -18 * np.abs(v)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((M, N), float("nan"), dtype=dtype, device=DEV)
        mx.gemm_mx(a, w, bias, out=out, activation=activation)
        within(out, want, bound + HALF[dtype] * (np.abs(want) + bound), f"{kind} -> {dtype}")


@pytest.mark.parametrize("kind", ["bfloat16", "mxfp8"])
@pytest.mark.parametrize("tile", [1, 2, 3, 4, 11, 12, 21, 22, 24, 41, 42, 44])
@pytest.mark.parametrize("M,N,K", [(1, 1, 8), (64, 64, 128), (129, 100, 136), (128, 128, 256), (257, 300, 1000), (300, 257, 384), (512, 520, 264)])
def test_tiles(mx, M, N, K, tile, kind):
    """Every tile at sizes inside it and past its edges, every epilogue. In the 2-norm what the scaled instruction cuts off stays below 1e-4: products have six
    significant bits, so only those under 2^-7 of their eight's largest lose any, a tenth of them at most, 2^-13 of it and a third of that in the mean."""
    w, wv = matrix(mx, N, K)
    a, av = rows_of(mx, M, K, kind)
    bias = rnd(N, seed=2)
    b = bias.double().cpu().numpy()
    want, bound = av @ wv.T + b, sums_bound(av, wv, b, K, kind == "mxfp8" and tile < 10)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((M + 3, N), float("nan"), dtype=dtype, device=DEV)
        mx.gemm_mx(a, w, bias, out=out[:M], shape=tile)
        within(out[:M], want, bound + HALF[dtype] * (np.abs(want) + bound), f"{kind} -> {dtype}")
        assert torch.isnan(out[M:]).all()
        if dtype == torch.float32:
            off = np.linalg.norm(out[:M].double().cpu().numpy() - want) / max(np.linalg.norm(av @ wv.T), 1e-30)
            assert off < (1e-4 if kind == "mxfp8" and tile < 10 else 1e-6), off
        act = torch.full((M, N), float("nan"), dtype=dtype, device=DEV)
        mx.gemm_mx(a, w, bias, out=act, activation="gelu_erf", shape=tile)
        exact = plain_mx.gelu(want, "gelu_erf")
        within(act, exact, 1.13 * bound + 2.0 ** -18 * np.abs(want) + HALF[dtype] * (np.abs(exact) + bound), "gelu_erf")
    stream = rnd(M, N, seed=3)
    before = stream.double().cpu().numpy()
    mx.gemm_mx(a, w, bias, residual=stream, shape=tile)
    within(stream, before + want, bound + HALF[torch.float32] * (np.abs(before) + np.abs(want) + bound), "residual")


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "mxfp8"])
@pytest.mark.parametrize("M", [1, 20, 70, 140])
def test_rows_that_are_no_numbers_stay_by_themselves(mx, M, kind):
    """A row of infinities or NaN makes its own results such and no other's; behind the row's end there is nothing, whatever memory holds there."""
    N, K = 40, 200
    w, wv = matrix(mx, N, K)
    if kind == "mxfp8":
        x = np.random.default_rng(5).normal(size=(M, K))
        x[M // 2, 7] = np.inf
        codes, scales = plain_mx.quantize(x, plain_mx.E4M3, 8)
        a, av = mx.Mxfp8Rows.pack(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV)), plain_mx.values(codes, scales, plain_mx.E4M3)
    else:
        wide = torch.full((M, K + 56), float("nan"), device=DEV, dtype=getattr(torch, kind))
        wide[:, :K] = rnd(M, K, dtype=getattr(torch, kind))
        wide[M // 2, 7] = float("inf")
        a = wide[:, :K]
        av = a.double().cpu().numpy()
    out = torch.zeros(M, N, device=DEV)
    mx.gemm_mx(a, w, None, out=out)
    others = [m for m in range(M) if m != M // 2]
    if others:
        within(out[others], av[others] @ wv.T, sums_bound(av[others], wv, np.zeros(N), K, kind == "mxfp8" and M > 64), kind)
    with np.errstate(invalid="ignore"):
        want = av[M // 2] @ wv.T
    got = out[M // 2].double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "mxfp8"])
def test_a_group_of_the_matrix_that_is_no_number(mx, kind):
    codes, scales = plain_mx.quantize(np.random.default_rng(0).normal(size=(20, 96)), plain_mx.E2M1, 2)
    scales[3, 1] = 255
    w = mx.Mxfp4Matrix.pack(torch.from_numpy(plain_mx.two_a_byte(codes)).to(DEV), torch.from_numpy(scales).to(DEV), 96)
    a, _ = rows_of(mx, 5, 96, kind)
    out = torch.zeros(5, 20, device=DEV)
    mx.gemm_mx(a, w, None, out=out)
    nan = torch.isnan(out).cpu()
    assert nan[:, 3].all() and not nan[:, :3].any() and not nan[:, 4:].any()


@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("M,K", [(3, 128), (70, 121), (140, 264)])
def test_rows_anywhere_in_memory(mx, M, K, shift, kind):
    """Rows that start between pieces of 16 bytes, with strides of any number of elements."""
    w, wv = matrix(mx, 50, K)
    dtype = getattr(torch, kind)
    flat = torch.full((M * (K + 5) + 16,), float("nan"), dtype=dtype, device=DEV)
    a = flat[shift:shift + M * (K + 5)].view(M, K + 5)[:, :K]
    a.copy_(rnd(M, K, dtype=dtype))
    av = a.double().cpu().numpy()
    out = torch.empty(M, 50, device=DEV)
    mx.gemm_mx(a, w, None, out=out)
    within(out, av @ wv.T, sums_bound(av, wv, np.zeros(50), K), kind)


def test_rows_far_apart(mx):
    """Rows whose places pass 32 bits: tiles, which find theirs by 32-bit offsets, are not chosen, and not taken."""
    from liyab_amd.errors import KernelError

    M, N, K, stride = 300, 256, 128, (1 << 22) + 8
    w, wv = matrix(mx, N, K)
    a = torch.empty(M * stride, dtype=torch.bfloat16, device=DEV).view(M, stride)[:, 64:64 + K]
    a.copy_(rnd(M, K, dtype=torch.bfloat16))
    av = a.double().cpu().numpy()
    out = torch.empty(M, N, device=DEV)
    mx.gemm_mx(a, w, None, out=out)
    within(out, av @ wv.T, sums_bound(av, wv, np.zeros(N), K), "far apart")
    with pytest.raises(KernelError):
        mx.gemm_mx(a, w, None, out=out, shape=1)


def test_scales_between_pieces_are_refused(mx):
    from liyab_amd.errors import KernelError

    codes, scales = mx.Mxfp8Rows.shapes(70, 256)
    flat = torch.zeros(70 * scales[1] + 16, dtype=torch.uint8, device=DEV)
    with pytest.raises(KernelError):
        mx.Mxfp8Rows(torch.zeros(codes, dtype=torch.uint8, device=DEV), flat[1:1 + 70 * scales[1]].view(scales), 256)


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "mxfp8"])
@pytest.mark.parametrize("M,H,Hkv,hd,K,page", [(1, 3, 3, 16, 64, 4), (33, 6, 3, 64, 128, 16), (20, 5, 1, 80, 1600, 16), (150, 4, 2, 32, 200, 48)])
def test_products_write_pages(mx, M, H, Hkv, hd, K, page, kind):
    """Queries to their rows, keys and values to their slots, and nothing anywhere else; a slot outside the pages is not written."""
    q_dim, kv_dim = H * hd, Hkv * hd
    N = q_dim + 2 * kv_dim
    w, _ = matrix(mx, N, K)
    a, _ = rows_of(mx, M, K, kind)
    bias = rnd(N, seed=2)
    dtype = torch.float32 if kind == "float32" else torch.bfloat16
    pages = -(-M // page) + 3
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(0))[:M].to(torch.int32).to(DEV)
    if M > 1:
        slots[1], slots[M - 1] = -1, pages * page
    flat = torch.empty(M, N, dtype=dtype, device=DEV)
    mx.gemm_mx(a, w, bias, out=flat)
    kc = torch.full((pages, Hkv, page, hd), 7.0, dtype=dtype, device=DEV)
    vc, q = kc.clone(), torch.zeros(M, q_dim, dtype=dtype, device=DEV)
    want_k, want_v = kc.clone(), vc.clone()
    mx.gemm_mx(a, w, bias, out=q, kv=(kc, vc, slots, q_dim))
    for m, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            want_k[s // page, :, s % page] = flat[m, q_dim:q_dim + kv_dim].view(Hkv, hd)
            want_v[s // page, :, s % page] = flat[m, q_dim + kv_dim:].view(Hkv, hd)
    assert torch.equal(q, flat[:, :q_dim]) and torch.equal(kc, want_k) and torch.equal(vc, want_v)


@pytest.mark.parametrize("M,N,K", [(40, 50, 320), (150, 264, 1000), (300, 520, 1664)])
@pytest.mark.parametrize("kind", ["bfloat16", "float32", "mxfp8"])
def test_rows_have_the_same_bits_among_others(mx, M, N, K, kind):
    """32-bit rows always, the others where the engine promises it."""
    from liyab_amd.kernels import ops

    w, _ = matrix(mx, N, K)
    a, _ = rows_of(mx, M, K, kind)

    def some_of(rows):
        if kind != "mxfp8":
            return a[rows]
        return mx.Mxfp8Rows(a.codes[rows].contiguous(), a.scales[rows].contiguous(), K)

    with ops.batch_invariant(kind != "float32"):
        out = torch.empty(M, N, device=DEV)
        mx.gemm_mx(a, w, None, out=out)
        for rows in (slice(0, 1), slice(7, 20), slice(3, 36), slice(M - 100, M - 1) if M > 140 else slice(1, 2)):
            part = torch.empty(rows.stop - rows.start, N, device=DEV)
            mx.gemm_mx(some_of(rows), w, None, out=part)
            assert torch.equal(part, out[rows])


# -- the formats ------------------------------------------------------------------------------------------------------


def hard_rows(n, d, seed=0, dtype=torch.float32):
    """Normal values, and groups of ties, of borders, of zeros, of the least and the largest numbers, of infinities and NaN."""
    x = torch.randn(n, d, generator=torch.Generator().manual_seed(seed)) * torch.logspace(-6, 6, n).unsqueeze(1)
    flat = x.view(-1)
    special = [1.75, 1.7500001, 448.0, 7.0, 7.0000005, 0.0, -0.0, 2.0 ** -149, 2.0 ** -127, 3.0e38, 1.0625, 1.1875, 0.25, -0.75, 2.5, 5.0, -6.5]
    for i, v in enumerate(special * 3):
        flat[(i * 37) % flat.numel()] = v
    if d > 64 and n > 2:
        x[1, 32:64] = 0.0
        x[2, 40], x[0, 33] = float("inf"), float("nan")
        x[n - 1, 32:64] = 2.0 ** -140
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 31), (4, 96), (5, 130), (17, 264), (40, 1000)])
def test_quantized_matrices_are_the_formats(mx, n, d, dtype):
    x = hard_rows(n, d, dtype=dtype)
    codes, scales = plain_mx.quantize(x.double().cpu().numpy(), plain_mx.E2M1, 2)
    want = plain_mx.values(codes, scales, plain_mx.E2M1)
    got = mx.Mxfp4Matrix.quantize(x)
    packed = mx.Mxfp4Matrix.pack(torch.from_numpy(plain_mx.two_a_byte(codes)).to(DEV), torch.from_numpy(scales).to(DEV), d)
    assert torch.equal(got.blocks, packed.blocks)
    dense = got.dense()
    assert np.array_equal(np.isnan(dense.cpu().numpy()), np.isnan(want))
    fine = ~np.isnan(want) & ((np.abs(want) >= 2.0 ** -126) & (np.abs(want) < 2.0 ** 128) | (want == 0))  # (32 bits hold less below, and not 4 times 2^126)
    assert np.array_equal(dense.double().cpu().numpy()[fine], want[fine])
    assert torch.equal(got.dense(torch.bfloat16).float().nan_to_num(5.0)[torch.from_numpy(fine)], dense.nan_to_num(5.0)[torch.from_numpy(fine)])


@pytest.mark.parametrize("n,d", [(3, 31), (5, 130), (196, 279), (16, 257), (4, 64)])
def test_packed_rows_of_whole_groups(mx, n, d):
    """Rows of codes may come as whole groups of 32; what lies behind the width does not count."""
    from liyab_amd.errors import KernelError

    g = torch.Generator().manual_seed(n * d)
    groups = -(-d // 32)
    codes = torch.randint(0, 256, (n, 16 * groups), generator=g, dtype=torch.uint8)
    scales = torch.randint(100, 140, (n, groups), generator=g, dtype=torch.uint8)
    plain = codes[:, : -(-d // 2)].clone()
    if d % 2:
        plain[:, -1] &= 15
    whole = mx.Mxfp4Matrix.pack(codes.to(DEV), scales.to(DEV), d)
    assert torch.equal(whole.blocks, mx.Mxfp4Matrix.pack(plain.to(DEV), scales.to(DEV), d).blocks)
    with pytest.raises(KernelError):
        mx.Mxfp4Matrix.pack(torch.zeros(n, 16 * groups + 1, dtype=torch.uint8, device=DEV), scales.to(DEV), d)


def check_rows(out, codes, scales, what):
    """Codes and bytes of rows, and zeros behind their width."""
    n, d = codes.shape
    got = out.codes.cpu().numpy()
    assert np.array_equal(got[:, :d], codes), f"{what}: {np.argwhere(got[:, :d] != codes)[:4].tolist()}"
    assert (got[:, d:] == 0).all(), f"{what}: behind the width"
    groups = scales.shape[1]
    assert np.array_equal(out.scales.cpu().numpy()[:, :groups], scales), what
    assert (out.scales.cpu().numpy()[:, groups:got.shape[1] // 32] == 0).all(), what


def empty_rows(mx, n, d):
    out = mx.Mxfp8Rows.empty(n, d, DEV)
    out.codes.fill_(0xAA)
    out.scales.fill_(0xAA)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 31), (4, 96), (5, 130), (17, 264), (9, 2050), (3, 5001)])
def test_rows_in_8_bits(mx, n, d, dtype):
    x = hard_rows(n, d, dtype=dtype)
    out = empty_rows(mx, n, d)
    mx.rows_mx(out, x)
    check_rows(out, *plain_mx.quantize(x.double().cpu().numpy(), plain_mx.E4M3, 8), "rows")
    wide = torch.full((n, d + 7), float("nan"), dtype=dtype, device=DEV)
    wide[:, 3:d + 3] = x
    again = empty_rows(mx, n, d)
    mx.rows_mx(again, wide[:, 3:d + 3])
    assert torch.equal(again.codes, out.codes)


def near_the_format(out, want, slack, what):
    """Rows in 8 bits against the exact values before rounding, known up to `slack`: a group's byte is that of its largest magnitude give or take the slack, and every
    number is off by half a step of its binade and the slack."""
    n, d = want.shape
    codes, scales = out.codes.cpu().numpy()[:, :d], out.scales.cpu().numpy()[:, : -(-d // 32)]
    assert (out.codes.cpu().numpy()[:, d:] == 0).all(), what
    got = plain_mx.values(codes, scales, plain_mx.E4M3)
    for i in range(n):
        for q in range(scales.shape[1]):
            part = slice(32 * q, min(32 * q + 32, d))
            mag = np.abs(want[i, part])
            low, high = plain_mx.scale_byte(max((mag - slack[i, part]).max(), 0.0), 8), plain_mx.scale_byte((mag + slack[i, part]).max(), 8)
            assert low <= scales[i, q] <= high, f"{what}: row {i}, group {q}: byte {scales[i, q]}, not {low} to {high}"
            unit = 2.0 ** (int(scales[i, q]) - 127)
            v = (mag + slack[i, part]) / unit
            half = 2.0 ** (np.floor(np.log2(np.maximum(v, 2.0 ** -6))) - 4) * unit
            off = np.abs(got[i, part] - want[i, part])
            assert (off <= half * (1 + 1e-9) + slack[i, part]).all(), f"{what}: row {i}, group {q}: {off.max()} of {half.max()}"


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh", "clamped"])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 33), (5, 128), (9, 200), (2, 2500)])
def test_gates(mx, n, d, activation):
    gu = rnd(n, 2 * d, seed=4, scale=3.0)
    g, u = gu.double().cpu().numpy()[:, :d], gu.double().cpu().numpy()[:, d:]
    out = empty_rows(mx, n, d)
    if activation == "clamped":
        limit, slope, shift = 2.5, 1.702, 1.0
        mx.glu_mx(out, gu, activation, clamp=(limit, slope, shift))
        g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
        want = g / (1 + np.exp(-slope * g)) * (u + shift)
        size = np.abs(g) * (np.abs(u) + shift)
    else:
        mx.glu_mx(out, gu, activation)
        want, size = plain_mx.gelu(g, activation) * u, np.abs(g * u)
    # an exponential whose argument (up to 2^6) is rounded, a reciprocal, three products, each of 32 bits
    near_the_format(out, want, 2.0 ** -17 * np.maximum(np.abs(want), 2.0 ** -6 * size), activation)
    wide = torch.full((n, 2 * d + 3), float("nan"), device=DEV)
    wide[:, 1:2 * d + 1] = gu
    again = empty_rows(mx, n, d)
    mx.glu_mx(again, wide[:, 1:2 * d + 1], activation, clamp=(2.5, 1.702, 1.0) if activation == "clamped" else None)
    assert torch.equal(again.codes, out.codes)


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh", "norm", "layer norm"])
def test_values_next_to_a_border_land_on_its_right_side(mx, kind):
    """A quarter of a million values as the definition in 64 bits rounds them. Both are off by less than 1e-9 of a value, two borders of a binade's 16 lie that close to one in 10^7
    of them: none, or this many values would say so about one seed in 40."""
    n, d = 64, 4096
    out = empty_rows(mx, n, d)
    if kind in ("silu", "gelu_tanh"):
        gu = rnd(n, 2 * d, seed=21)
        mx.glu_mx(out, gu, kind)
        v = gu.double().cpu().numpy()
        y = plain_mx.gelu(v[:, :d], kind) * v[:, d:]
    else:
        x, add, w, b = rnd(n, d, seed=22), rnd(n, d, seed=23), 1 + 0.3 * rnd(d, seed=24), rnd(d, seed=25, scale=0.2)
        mx.norm_mx(out, x, w, 0.0, bias=b, centred=kind == "layer norm", add=add)
        t = x.double().cpu().numpy() + add.double().cpu().numpy()
        t = t - (t.mean(axis=1, keepdims=True) if kind == "layer norm" else 0.0)
        y = t / np.sqrt((t ** 2).mean(axis=1, keepdims=True)) * w.double().cpu().numpy() + b.double().cpu().numpy()
    check_rows(out, *plain_mx.quantize(y, plain_mx.E4M3, 8), kind)


@pytest.mark.parametrize("centred", [False, True])
@pytest.mark.parametrize("added", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 40), (4, 130), (3, 512), (5, 513), (7, 1600), (2, 2049), (2, 4100), (2, 8200), (1, 20000), (2, 40003)])
def test_norms(mx, n, d, added, centred):
    """Sums of d squares in 32 bits: a lane's up to 64 in a chain, then the lanes' and waves' trees: 100 roundings at most, half of them under the root; the mean likewise."""
    x = rnd(n, d, seed=5) * torch.logspace(-2, 2, n, device=DEV).unsqueeze(1) + 0.25
    add = None if added is None else rnd(n, d, seed=6, dtype=added)
    w, b = 1 + 0.3 * rnd(d, seed=7), rnd(d, seed=8, scale=0.2)
    t = x if add is None else x + add.float()
    tv = t.double().cpu().numpy()
    mean = tv.mean(axis=1, keepdims=True) if centred else np.zeros((n, 1))
    r = 1 / np.sqrt(((tv - mean) ** 2).mean(axis=1, keepdims=True) + 1e-5)
    wv, bv = w.double().cpu().numpy(), b.double().cpu().numpy()
    slack = 100 * 2.0 ** -24 * ((np.abs(tv) + np.abs(mean) + np.abs(tv).mean(axis=1, keepdims=True) * centred) * r * np.abs(wv) + np.abs(bv) * centred) + 1e-30
    # (a row's own deviation: what the mean's error does to the squares under the root)
    slack *= 1 + np.abs(mean) * r
    for out_stream in (None, torch.empty_like(x)):
        out = empty_rows(mx, n, d)
        mx.norm_mx(out, x, w, 1e-5, bias=b if centred else None, centred=centred, add=add, stream=out_stream)
        near_the_format(out, (tv - mean) * r * wv + (bv if centred else 0.0), slack, f"centred {centred}")
        if out_stream is not None:
            assert torch.equal(out_stream, t)
    inplace, again = x.clone(), empty_rows(mx, n, d)
    mx.norm_mx(again, inplace, w, 1e-5, bias=b if centred else None, centred=centred, add=add, stream=inplace)
    assert torch.equal(inplace, t) and torch.equal(again.codes, out.codes) and torch.equal(again.scales[:, : -(-d // 32)], out.scales[:, : -(-d // 32)])


def test_norms_of_rows_that_are_no_numbers(mx):
    """A row with an infinity has no norm; zeros have one, and their neighbours theirs."""
    x = rnd(4, 200, seed=5)
    x[1, 3], x[2] = float("inf"), 0.0
    out = empty_rows(mx, 4, 200)
    mx.norm_mx(out, x, None, 1e-5)
    scales = out.scales.cpu().numpy()[:, :7]
    assert scales[1, 0] == 255 and (scales[[0, 2, 3]] < 255).all() and (out.codes[2] == 0).all()
    assert (out.codes.cpu().numpy()[:, 200:] == 0).all()


# -- refusals -----------------------------------------------------------------------------------------------------------


def test_refusals(mx):
    from liyab_amd.errors import KernelError

    w, _ = matrix(mx, 32, 64)
    a, out = rnd(4, 64, dtype=torch.bfloat16), torch.empty(4, 32, device=DEV)
    rows = mx.Mxfp8Rows.empty(4, 64)
    bad = [
        lambda: mx.gemm_mx(rnd(4, 65, dtype=torch.bfloat16), w, None, out=out),
        lambda: mx.gemm_mx(a.half(), w, None, out=out),
        lambda: mx.gemm_mx(a.cpu(), w, None, out=out),
        lambda: mx.gemm_mx(a.t(), w, None, out=out),
        lambda: mx.gemm_mx(a, w, None, out=out[:3]),
        lambda: mx.gemm_mx(a, w, None),
        lambda: mx.gemm_mx(a, w, rnd(31), out=out),
        lambda: mx.gemm_mx(a, w, None, residual=out.bfloat16()),
        lambda: mx.gemm_mx(mx.Mxfp8Rows.empty(4, 96), w, None, out=out),
        lambda: mx.rows_mx(rows, rnd(4, 65)),
        lambda: mx.rows_mx(rows, rnd(3, 64)),
        lambda: mx.rows_mx(rows, rnd(4, 64).half()),
        lambda: mx.glu_mx(rows, rnd(4, 64), "silu"),
        lambda: mx.glu_mx(rows, rnd(4, 128), "relu"),
        lambda: mx.glu_mx(rows, rnd(4, 128), "clamped"),
        lambda: mx.glu_mx(rows, rnd(4, 128), "clamped", clamp=(0.0, 1.0, 0.0)),
        lambda: mx.glu_mx(rows, rnd(4, 128, dtype=torch.bfloat16), "silu"),
        lambda: mx.norm_mx(rows, rnd(4, 64, dtype=torch.bfloat16), None, 1e-5),
        lambda: mx.norm_mx(rows, rnd(4, 128)[:, :64], None, 1e-5),
        lambda: mx.norm_mx(rows, rnd(4, 64), rnd(63), 1e-5),
        lambda: mx.norm_mx(rows, rnd(4, 64), None, 1e-5, add=rnd(3, 64)),
        lambda: mx.norm_mx(rows, rnd(4, 64), None, 1e-5, stream=rnd(4, 64, dtype=torch.bfloat16)),
        lambda: mx.norm_mx(mx.Mxfp8Rows.empty(1, 65537), rnd(1, 65537), None, 1e-5),
        lambda: mx.Mxfp4Matrix.quantize(rnd(4, 64).half()),
        lambda: mx.Mxfp4Matrix.pack(torch.zeros(4, 32, dtype=torch.uint8, device=DEV), torch.zeros(4, 3, dtype=torch.uint8, device=DEV), 64),
        lambda: mx.Mxfp4Matrix(w.blocks, 32, 200),
        lambda: mx.Mxfp4Matrix(w.blocks.view(-1)[1:1 + 2 * 1088].view(2, 1, 1088), 32, 64) if w.blocks.numel() > 2 * 1088 else mx.Mxfp4Matrix(w.blocks, 33, 64),
        lambda: mx.Mxfp8Rows(rows.codes[:, :64], rows.scales, 64),
        lambda: mx.Mxfp8Rows(rows.codes, rows.scales[:2], 64),
        lambda: mx.Mxfp8Rows.pack(torch.zeros(4, 64, device=DEV), torch.zeros(4, 2, dtype=torch.uint8, device=DEV)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(KernelError):
            call()
            pytest.fail(f"call {i} was taken")


def test_no_rows(mx):
    w, _ = matrix(mx, 32, 64)
    mx.gemm_mx(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV), w, None, out=torch.empty(0, 32, device=DEV))
    none = mx.Mxfp8Rows.empty(0, 64)
    mx.rows_mx(none, torch.empty(0, 64, device=DEV))
    mx.glu_mx(none, torch.empty(0, 128, device=DEV), "silu")
    mx.norm_mx(none, torch.empty(0, 64, device=DEV), None, 1e-5)
    mx.gemm_mx(none, w, None, out=torch.empty(0, 32, device=DEV))


# -- together -------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("n", [1, 9, 150])
def test_a_gated_feed_forward_in_a_graph_and_on_another_stream(mx, n):
    """norm -> [gate | up] -> gate -> down, added to the stream: eager, on a stream of its own, and replayed from a graph with new rows, the same bits each time; the last
    product against float64 of the rows that it read."""
    d, ff = 192, 328
    w1, _ = matrix(mx, 2 * ff, d, seed=1)
    w2, w2v = matrix(mx, d, ff, seed=2)
    nw = 1 + 0.2 * rnd(d, seed=3)
    x, y = torch.empty(n, d, device=DEV), torch.empty(n, d, device=DEV)
    h, inner, gu = mx.Mxfp8Rows.empty(n, d), mx.Mxfp8Rows.empty(n, ff), torch.empty(n, 2 * ff, device=DEV)

    def run():
        mx.norm_mx(h, x, nw, 1e-5, add=y, stream=x)
        mx.gemm_mx(h, w1, None, out=gu)
        mx.glu_mx(inner, gu, "silu")
        mx.gemm_mx(inner, w2, None, residual=x)

    def fill(seed):
        x.copy_(rnd(n, d, seed=seed))
        y.copy_(rnd(n, d, seed=seed + 1))

    def eager(seed):
        fill(seed)
        run()
        torch.cuda.synchronize()
        return x.clone()

    want = [eager(10), eager(20)]
    rows = plain_mx.values(inner.codes.cpu().numpy()[:, :ff], inner.scales.cpu().numpy()[:, : -(-ff // 32)], plain_mx.E4M3)
    before = (rnd(n, d, seed=20) + rnd(n, d, seed=21)).double().cpu().numpy()
    within(want[1], before + rows @ w2v.T, sums_bound(rows, w2v, np.zeros(d), ff, n > 64) + 2.0 ** -23 * (np.abs(before) + np.abs(rows @ w2v.T)), "down")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fill(10)
        run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(x, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed, expected in ((10, want[0]), (20, want[1]), (10, want[0])):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, expected)


# -- sums ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("shape", [0, 1, 2, 3, 4, 44])
@pytest.mark.parametrize("M,N,K", [(65, 40, 128), (130, 257, 392), (300, 512, 1000)])
def test_rows_in_8_bits_sum_in_32_bits(mx, M, N, K, shape):
    """Eight neighbours of every row hold two that cancel beside six that lie up to 2^-15 below them, and the result is those six and the row's others. Their products are whole
    multiples of 2^-8 and no partial sum reaches 2^13: 32 bits hold all of them, and nothing is off. Random rows are off by less than 2^-24 sqrt(K) in the 2-norm: a rounding
    of 2^-25 of the sum in the mean at each of fewer than K additions that do not know of each other."""
    rng = np.random.default_rng(M)
    codes = np.zeros((M, K), dtype=np.uint8)
    low = 8 + np.arange(1, 33)  # 2^-6 to 2^-2
    codes[:] = rng.choice(low, size=(M, K)) | (128 * rng.integers(0, 2, size=(M, K))).astype(np.uint8)
    at = rng.integers(0, K // 8, size=M) * 8
    codes[np.arange(M), at], codes[np.arange(M), at + 1] = 126, 126 | 128  # 448 and -448
    scales = np.full((M, -(-K // 32)), 127, dtype=np.uint8)
    wc = np.repeat(7 | (8 * rng.integers(0, 2, size=(N, -(-K // 8)))), 8, axis=1)[:, :K].astype(np.uint8)  # 6 or -6, eight of a sign
    ws = np.full((N, -(-K // 32)), 127, dtype=np.uint8)
    w = mx.Mxfp4Matrix.pack(torch.from_numpy(plain_mx.two_a_byte(wc)).to(DEV), torch.from_numpy(ws).to(DEV), K)
    a = mx.Mxfp8Rows.pack(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV))
    av, wv = plain_mx.values(codes, scales, plain_mx.E4M3), plain_mx.values(wc, ws, plain_mx.E2M1)
    out = torch.empty(M, N, device=DEV)
    mx.gemm_mx(a, w, None, out=out, shape=shape)
    assert np.array_equal(out.double().cpu().numpy(), av @ wv.T)
    w, wv = matrix(mx, N, K)
    a, av = rows_of(mx, M, K, "mxfp8")
    mx.gemm_mx(a, w, None, out=out, shape=shape)
    want = av @ wv.T
    assert np.linalg.norm(out.double().cpu().numpy() - want) < 2.0 ** -24 * K ** 0.5 * np.linalg.norm(want)


def beside_borders(c, seed):
    """Weights that put c / rms(c) of a row next to borders of e4m3, as near as 32 bits can say them (a few 2^-26 of a value); 400, and with it the groups' scale, in every 32nd place."""
    rng = np.random.default_rng(seed)
    d = c.size
    v = (8 + rng.integers(0, 8, size=d) + 0.5) * np.exp2(rng.integers(-3, 8, size=d) - 3.0)
    v[::32] = 400.0
    return (v / (np.abs(c) / np.sqrt((c ** 2).mean()))).astype(np.float32)


@pytest.mark.parametrize("centred", [False, True])
@pytest.mark.parametrize("to", ["nowhere", "beside", "x"])
@pytest.mark.parametrize("d", [1600, 16384, 20000])
def test_norms_next_to_borders_whatever_the_width_and_the_stream(mx, d, to, centred):
    """x + add is not rounded ahead of the norm, whether the stream is written or not, and where: a rounding to 32 bits would move values by up to 2^-24 of them across borders that lie nearer.
    In 64 bits both sides are off by some 1e-15: one of these values in 10^7 lies that close."""
    x, add = rnd(1, d, seed=31), rnd(1, d, seed=32)
    t = x.double().cpu().numpy() + add.double().cpu().numpy()
    c = t - t.mean() if centred else t
    w = torch.from_numpy(beside_borders(c[0], 33)).to(DEV)
    out = empty_rows(mx, 1, d)
    stream = {"nowhere": None, "beside": torch.empty_like(x), "x": x}[to]
    want = x + add
    mx.norm_mx(out, x, w, 0.0, centred=centred, add=add, stream=stream)
    y = c / np.sqrt((c ** 2).mean()) * w.double().cpu().numpy()
    check_rows(out, *plain_mx.quantize(y, plain_mx.E4M3, 8), to)
    assert stream is None or torch.equal(stream, want)


def test_what_gates_and_norms_are_given_is_taken_in_64_bits(mx):
    """A slope and a shift that 32 bits do not hold, and an eps as large as the squares, over values beside borders that the rounded numbers would put on the other side. Gates are off by
    up to 6e-11 of a value: those that lie nearer than 1e-9 of it to a border are left out."""
    rng = np.random.default_rng(41)
    limit, slope, shift = 6.7, 1.702, 1.1

    def gate(g, u, slope, shift):
        g = np.minimum(g, limit)
        return g / (1 + np.exp(-slope * g)) * (np.clip(u, -limit, limit) + shift)

    def place(v):  # among the borders of numbers with three bits of mantissa
        e = np.floor(np.log2(np.abs(v)))
        return 8 * e + np.floor((np.abs(v) * np.exp2(-e) * 16 + 1) / 2)

    g = rng.uniform(0.5, 3.0, size=1 << 14).astype(np.float32).astype(np.float64)
    border = (8 + rng.integers(0, 8, size=g.size) + 0.5) * np.exp2(rng.integers(-2, 4, size=g.size) - 3.0)
    u = (border / gate(g, 1.0 - shift, slope, shift) - shift).astype(np.float32).astype(np.float64)
    y, low = gate(g, u, slope, shift), gate(g, u, float(np.float32(slope)), float(np.float32(shift)))
    near = np.flatnonzero((np.abs(u) < 6) & (place(y) != place(low)) & (place(y * (1 - 1e-9)) == place(y * (1 + 1e-9))))
    n = near.size // 31
    assert n > 20
    g, u = (np.concatenate([np.full((n, 1), b), v[near[:31 * n]].reshape(n, 31)], axis=1) for b, v in ((6.0, g), (9.0, u)))  # (6 and 9, a gate of 46.8: the groups' scale)
    out = empty_rows(mx, n, 32)
    mx.glu_mx(out, torch.from_numpy(np.concatenate([g, u], axis=1)).float().to(DEV), "clamped", clamp=(limit, slope, shift))
    check_rows(out, *plain_mx.quantize(gate(g, u, slope, shift), plain_mx.E4M3, 8), "clamped")

    x, eps = rnd(1, 4096, seed=42, scale=0.01), 1e-4
    v = x.double().cpu().numpy()
    c = v / np.sqrt((v ** 2).mean() + eps)
    w = torch.from_numpy((beside_borders(v[0], 43).astype(np.float64) * (v / np.sqrt((v ** 2).mean()) / c)[0]).astype(np.float32)).to(DEV)
    out = empty_rows(mx, 1, 4096)
    mx.norm_mx(out, x, w, eps)
    check_rows(out, *plain_mx.quantize(c * w.double().cpu().numpy(), plain_mx.E4M3, 8), "norm")


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh", "clamped"])
def test_gates_of_what_is_no_number(mx, activation):
    """A NaN in either half makes its group no number, and no other; an infinity does where nothing clamps it."""
    d, clamp = 200, (2.5, 1.702, 1.0) if activation == "clamped" else None
    gu = rnd(6, 2 * d, seed=51)
    plain = empty_rows(mx, 6, d)
    mx.glu_mx(plain, gu, activation, clamp=clamp)
    gu[0, 40] = gu[1, d + 70] = gu[2, 199] = gu[2, 2 * d - 1] = float("nan")
    gu[3, 33], gu[4, d + 33] = float("inf"), float("-inf")
    out = empty_rows(mx, 6, d)
    mx.glu_mx(out, gu, activation, clamp=clamp)
    scales = out.scales.cpu().numpy()[:, :7]
    no_number = np.zeros((6, 7), dtype=bool)
    no_number[0, 1] = no_number[1, 2] = no_number[2, 6] = True
    no_number[3, 1] = no_number[4, 1] = activation != "clamped"
    assert np.array_equal(scales == 255, no_number)
    same = ~np.repeat(no_number, 32, axis=1)[:, :d]
    same[3:5, 32:64] = False
    assert np.array_equal(out.codes.cpu().numpy()[:, :d][same], plain.codes.cpu().numpy()[:, :d][same])
    if activation == "clamped":  # what lies beyond the limits is the limit
        gu[3, 33], gu[4, d + 33] = 2.5, -2.5
        for i in range(3):
            gu[i] = 0.0
        again = empty_rows(mx, 6, d)
        mx.glu_mx(again, gu, activation, clamp=clamp)
        assert torch.equal(again.codes[3:], out.codes[3:])


def test_calls_that_say_two_things_are_refused(mx):
    """Nothing that a call says is left out in silence, and nothing of it is done where it is refused."""
    from liyab_amd.errors import KernelError

    w, _ = matrix(mx, 32, 64)
    a, wide = rnd(4, 64, dtype=torch.bfloat16), rnd(4, 64)
    out, stream, rows = torch.zeros(4, 32, device=DEV), torch.zeros(4, 32, device=DEV), mx.Mxfp8Rows.empty(4, 64)
    kc = torch.zeros(2, 1, 16, 8, dtype=torch.bfloat16, device=DEV)
    q, vc, slots = torch.zeros(4, 16, dtype=torch.bfloat16, device=DEV), kc.clone(), torch.arange(4, dtype=torch.int32, device=DEV)
    bad = [
        lambda: mx.gemm_mx(a, w, None, residual=stream, activation="gelu_tanh"),
        lambda: mx.gemm_mx(a, w, None, residual=stream, out=out),
        lambda: mx.gemm_mx(a, w, None, residual=stream, kv=(kc, vc, slots, 16)),
        lambda: mx.gemm_mx(a, w, None, out=q, kv=(kc, vc, slots, 16), activation="gelu_erf"),
        lambda: mx.gemm_mx(a, w, None, out=out, activation="relu"),
        lambda: mx.gemm_mx(a, w, None, out=out, activation=None),
        lambda: mx.gemm_mx(wide, w, None, out=out, shape=1),
        lambda: mx.gemm_mx(a, w, None, out=out, shape=5),
        lambda: mx.gemm_mx(a, rnd(32, 64, dtype=torch.bfloat16), None, out=out),
        lambda: mx.rows_mx(out, wide),
        lambda: mx.norm_mx(out, wide, None, 1e-5),
        lambda: mx.glu_mx(out, rnd(4, 128), "silu"),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(KernelError):
            call()
            pytest.fail(f"call {i} was taken")
    for t in (out, stream, q, kc, vc):
        assert not t.any()
    mx.gemm_mx(a, w, None, out=q, kv=(kc, vc, slots, 16))
    assert q.any() and kc.any() and vc.any()


@pytest.mark.parametrize("d", [64, 300, 20000])
def test_the_stream_is_what_the_norm_reads_or_lies_apart(mx, d):
    """x and add may be the stream, value by value; a stream that lies across either of them would be read where another row has written."""
    from liyab_amd.errors import KernelError

    n, w = 3, 1 + 0.2 * rnd(d, seed=61)
    x, add = rnd(n, d, seed=62), rnd(n, d, seed=63)
    want, stream = mx.Mxfp8Rows.empty(n, d), torch.empty(n, d, device=DEV)
    mx.norm_mx(want, x, w, 1e-5, add=add, stream=stream)
    for which in ("x", "add"):
        a, b, out = x.clone(), add.clone(), mx.Mxfp8Rows.empty(n, d)
        mx.norm_mx(out, a, w, 1e-5, add=b, stream=a if which == "x" else b)
        assert torch.equal(a if which == "x" else b, stream) and torch.equal(out.codes, want.codes) and torch.equal(out.scales[:, : d // 32], want.scales[:, : d // 32])
    flat = torch.zeros((n + 1) * d, device=DEV)
    low, high = flat[: n * d].view(n, d), flat[d:].view(n, d)
    half = flat.view(torch.bfloat16)[: n * d].view(n, d)
    for kw in (dict(x=low, stream=high), dict(x=high, stream=low), dict(x=x, add=low, stream=high), dict(x=x, add=half, stream=low)):
        with pytest.raises(KernelError):
            mx.norm_mx(want, kw.pop("x"), w, 1e-5, **kw)
    assert not flat.any()


@pytest.mark.parametrize("added", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [33, 512, 513, 2049, 4100, 8200, 40003])
def test_norms_next_to_borders_at_every_kernel_and_odd_widths(mx, d, added):
    """Sums of 32 bits anywhere in a norm would put some of these values on the wrong side of a border: they lie a few 2^-26 beside one."""
    x, add = rnd(1, d, seed=71), rnd(1, d, seed=72, dtype=added)
    t = x.double().cpu().numpy() + add.double().cpu().numpy()
    for centred in (False, True):
        c = t - t.mean() if centred else t
        w = torch.from_numpy(beside_borders(c[0], 73)).to(DEV)
        out = empty_rows(mx, 1, d)
        mx.norm_mx(out, x, w, 0.0, centred=centred, add=add)
        check_rows(out, *plain_mx.quantize(c / np.sqrt((c ** 2).mean()) * w.double().cpu().numpy(), plain_mx.E4M3, 8), f"centred {centred}")


@pytest.mark.parametrize("activation", ["silu", "gelu_tanh", "clamped"])
@pytest.mark.parametrize("n,d", [(7, 33), (3, 514), (2, 2500), (5, 4096)])
def test_gates_next_to_borders(mx, n, d, activation):
    """Values within 2^-24 of a border, and further than the 1e-9 that a gate's exponential and quotient stay well below."""
    rng = np.random.default_rng(81)
    slope, shift, limit = 1.75, 0.5, 1024.0  # (32 bits hold these)
    g = rng.uniform(0.5, 4.0, size=(n, d)).astype(np.float32).astype(np.float64)
    a = plain_mx.gelu(g, activation) if activation != "clamped" else g / (1 + np.exp(-slope * g))
    shift = shift if activation == "clamped" else 0.0
    border = (8 + rng.integers(0, 8, size=(n, d)) + 0.5) * np.exp2(rng.integers(-3, 8, size=(n, d)) - 3.0)
    border[:, ::32] = 400.0
    u = (border / a - shift).astype(np.float32)
    near = np.abs(a * (u.astype(np.float64) + shift) / border - 1) < 1e-9
    u[near] = np.nextafter(u[near], np.float32(2000))
    u = u.astype(np.float64)
    out = empty_rows(mx, n, d)
    mx.glu_mx(out, torch.from_numpy(np.concatenate([g, u], axis=1)).float().to(DEV), activation, clamp=(limit, slope, shift) if activation == "clamped" else None)
    u = np.clip(u, -limit, limit) if activation == "clamped" else u
    check_rows(out, *plain_mx.quantize(a * (u + shift), plain_mx.E4M3, 8), activation)


def test_blocks_between_pieces_are_refused(mx):
    """Blocks start on 16-byte boundaries, as the products' loads take them."""
    from liyab_amd.errors import KernelError

    flat = torch.zeros(2 * mx.BLOCK_BYTES + 16, dtype=torch.uint8, device=DEV)
    mx.Mxfp4Matrix(flat[16:].view(2, 1, mx.BLOCK_BYTES), 32, 64)
    for at in (1, 4, 8, 15):
        with pytest.raises(KernelError):
            mx.Mxfp4Matrix(flat[at:at + 2 * mx.BLOCK_BYTES].view(2, 1, mx.BLOCK_BYTES), 32, 64)


def test_packed_numbers_are_of_the_formats_types(mx):
    """Bytes, or torch's types of the same numbers; other 8-bit types hold other numbers in the same bytes."""
    from liyab_amd.errors import KernelError

    g = torch.Generator().manual_seed(91)
    codes = (torch.randint(0, 126, (3, 64), generator=g, dtype=torch.uint8) + 128 * torch.randint(0, 2, (3, 64), generator=g, dtype=torch.uint8)).to(DEV)
    four, scales = torch.randint(0, 256, (3, 32), generator=g, dtype=torch.uint8).to(DEV), torch.randint(100, 140, (3, 2), generator=g, dtype=torch.uint8).to(DEV)
    rows = mx.Mxfp8Rows.pack(codes, scales)
    typed = mx.Mxfp8Rows.pack(codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu))
    assert torch.equal(rows.codes, typed.codes) and torch.equal(rows.scales, typed.scales)
    matrix = mx.Mxfp4Matrix.pack(four, scales, 64)
    assert torch.equal(matrix.blocks, mx.Mxfp4Matrix.pack(four.view(torch.float4_e2m1fn_x2), scales.view(torch.float8_e8m0fnu), 64).blocks)
    for other in (torch.float8_e5m2, torch.float8_e4m3fnuz, torch.float8_e5m2fnuz, torch.float8_e8m0fnu, torch.int8, torch.float4_e2m1fn_x2):
        with pytest.raises(KernelError):
            mx.Mxfp8Rows.pack(codes.view(other), scales)
    for other in (torch.float8_e4m3fn, torch.float8_e5m2, torch.int8):
        with pytest.raises(KernelError):
            mx.Mxfp4Matrix.pack(four.view(other), scales, 64)
        with pytest.raises(KernelError):
            mx.Mxfp8Rows.pack(codes, scales.view(other))
        with pytest.raises(KernelError):
            mx.Mxfp4Matrix.pack(four, scales.view(other), 64)
