"""Every tile shape of the products on rows sorted by expert, sums that begin inside the row, and the tiled kernels among
NaN neighbours, in a captured graph, on two streams and called twice.

Each case asserts the shape that it is for.  (Of TILES in test_gpu_products, "256x128", "128x128" and "128x64" take tiles of
128 x 64 under the launcher's rule, and no forward product there takes tiles of 128 columns.)"""
import pytest
import torch

import products_ref as ref

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
OUT = [torch.bfloat16, torch.float16, torch.float32]
FEW_WORK = 3 << 29   # rows * columns * bytes of a weight row up to which the few-rows kernel runs


def tile_shape(M, P, R, E, bytes_):
    """The tile (rows, columns) that the launcher takes for M rows, P columns and sums of R; E 0: one weight for all rows."""
    if M * P * R <= FEW_WORK // bytes_:
        return None
    best, most = (256, 256), 0
    for rows, cols in ((256, 256), (256, 128), (128, 128), (256, 64), (128, 64)):
        groups, whole = min(M, E), M // rows
        items = max(groups, whole + groups // 2) if E else -(-M // rows)
        tiles = items * -(-P // cols)
        if most < tiles <= 256:
            best, most = (rows, cols), tiles
    return best


def _say(*a):
    print(*a, flush=True)


def _starts(counts, head=0):
    s = [head]
    for c in counts:
        s.append(s[-1] + c)
    return torch.tensor(s, dtype=torch.int32)


def _rand(cuda, dt, seed, *shapes):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(*s, generator=g, device=cuda).to(dt) for s in shapes]


def _codes(cuda, seed, *shapes):
    """Codes of the whole range, and scales that keep outputs far below fp16's largest."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for s in shapes:
        out.append(torch.randint(-128, 128, s, generator=g, device=cuda, dtype=torch.int32).to(torch.int8))
        out.append(torch.rand(s[:-1], generator=g, device=cuda) * 0.001 + 1e-5)
    return out


# tile: rows of each expert, rows before the first and behind the last, columns, sum (16 bits; int8 takes twice that).  Sums
# of whole lines of 128 bytes, which may begin inside the row, and others.
GROUPED = [((256, 256), [300] * 9, 1, 7, 3500, 264), ((256, 256), [40, 120, 64, 1, 0, 128] * 3, 2, 3, 2060, 576),
           ((256, 128), [40, 64, 0, 128, 3, 65, 20, 90] * 2, 0, 5, 1544, 1280), ((256, 128), [150, 30, 60, 10] * 4, 3, 0, 1537, 1000),
           ((128, 128), [1000], 0, 0, 3001, 320), ((128, 128), [997], 0, 3, 3000, 328),
           ((256, 64), [33, 70, 140, 0] * 3, 0, 0, 1280, 2048), ((256, 64), [33] * 12, 1, 2, 1277, 1992),
           ((128, 64), [400], 0, 3, 1000, 2112), ((128, 64), [513], 0, 0, 2040, 1608)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(GROUPED)))
def test_shapes_16bit(cuda, dt, case):
    """Rows along the sum (y), and across it (dx)."""
    tile, counts, head, tail, P, R = GROUPED[case]
    M, E, t = head + sum(counts) + tail, len(counts), DT[dt]
    assert tile_shape(M, P, R, E, 2) == tile
    s = _starts(counts, head)
    x, w = _rand(cuda, t, P + R, (M, R), (E, P, R))
    _say("[shapes]", tile, M, P, R, E, t)
    ops = torch.ops.nanovllm
    y = ops.moe_grouped_matmul(x, w, s.to(cuda))
    assert ref.within(y, *ref.grouped(x, w, s.tolist(), t)) <= 1.0
    assert torch.equal(y, ops.moe_grouped_matmul(x, w, s.to(cuda)))
    P8 = P // 8 * 8   # the columns of dx are a row's length
    w = w[:, :P8].transpose(1, 2).contiguous()
    assert tile_shape(M, P8, R, E, 2) == tile
    dx = ops.moe_grouped_matmul_dx(x, w, s.to(cuda))
    assert ref.within(dx, *ref.grouped_dx(x, w, s.tolist(), t)) <= 1.0
    assert torch.equal(dx, ops.moe_grouped_matmul_dx(x, w, s.to(cuda)))


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("case", range(len(GROUPED)))
def test_shapes_int8_grouped(cuda, out, case):
    tile, counts, head, tail, P, R = GROUPED[case]
    M, E, R = head + sum(counts) + tail, len(counts), 2 * R
    assert tile_shape(M, P, R, E, 1) == tile
    s = _starts(counts, head)
    x, xs, w, ws = _codes(cuda, P + R, (M, R), (E, P, R))
    _say("[shapes int8]", tile, M, P, R, E, out)
    ops = torch.ops.nanovllm
    y = ops.moe_grouped_matmul_int8(x, xs, w, ws, s.to(cuda), out)
    assert ref.within(y, *ref.int8_grouped(x, xs, w, ws, s.tolist(), out)) <= 1.0
    assert torch.equal(y, ops.moe_grouped_matmul_int8(x, xs, w, ws, s.to(cuda), out))


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("tile,M,N,K", [((256, 256), 2000, 6001, 272), ((256, 128), 200, 19001, 2048), ((256, 128), 131, 20000, 1040),
                                        ((128, 128), 1000, 2100, 1024), ((256, 64), 128, 16001, 1040), ((128, 64), 333, 1001, 8208)])
def test_shapes_int8_dense(cuda, out, tile, M, N, K):
    assert tile_shape(M, N, K, 0, 1) == tile
    x, xs, w, ws = _codes(cuda, N + K, (M, K), (N, K))
    bias = torch.randn(N, generator=torch.Generator(device="cuda").manual_seed(N), device=cuda)
    _say("[shapes int8 dense]", tile, M, N, K, out)
    y = torch.ops.nanovllm.int8_matmul(x, xs, w, ws, bias, out)
    assert ref.within(y, *ref.int8_rows(x, xs, w, ws, bias, out)) <= 1.0


# Sums that may begin inside the row, several tiles a workgroup: rows of each expert
WRAPPED = {"up to 64": [16, 1, 33, 0, 64, 20, 7, 63], "up to 128": [65, 128, 100, 81, 97, 127, 70, 90],
           "mixed": [10, 0, 64, 65, 128, 129, 200, 3]}


@pytest.mark.parametrize("kind", ["bf16", "fp16", "int8"])
@pytest.mark.parametrize("name", WRAPPED)
def test_wrapped_sums(cuda, kind, name):
    counts, N, K, ops = WRAPPED[name] * 16, 1536, 512, torch.ops.nanovllm
    E, M, s = len(counts), sum(counts) + 4, _starts(counts, 1)
    _say("[wrapped]", name, kind, M)
    if kind == "int8":
        K = 1024
        assert tile_shape(M, N, K, E, 1) == (256, 256)
        x, xs, w, ws = _codes(cuda, M, (M, K), (E, N, K))
        y = ops.moe_grouped_matmul_int8(x, xs, w, ws, s.to(cuda), torch.float32)
        assert ref.within(y, *ref.int8_grouped(x, xs, w, ws, s.tolist(), torch.float32)) <= 1.0
    else:
        assert tile_shape(M, N, K, E, 2) == (256, 256)
        x, w = _rand(cuda, DT[kind], M, (M, K), (E, N, K))
        y = ops.moe_grouped_matmul(x, w, s.to(cuda))
        assert ref.within(y, *ref.grouped(x, w, s.tolist(), DT[kind])) <= 1.0


# The tiled kernels as the small calls of the other tests are checked: rows of each expert, N, K
TILED = [([300, 0, 200], 2056, 1640), ([30, 0, 100, 64] * 4, 1544, 1536)]


@pytest.mark.parametrize("counts,N,K", TILED)
def test_tiled_neighbours_do_not_leak(cuda, counts, N, K):
    """NaN and infinities in rows of no expert and in unused experts' weights stay there; so does those of one row."""
    ops, E, M = torch.ops.nanovllm, len(counts), sum(counts) + 9
    s = _starts(counts, head=2).to(cuda)
    x, w, dy = _rand(cuda, torch.bfloat16, N, (M, K), (E, N, K), (M, N))
    assert tile_shape(M, N, K, E, 2) and tile_shape(M, K, N, E, 2)
    x2, w2, dy2 = x.clone(), w.clone(), dy.clone()
    x2[:2], x2[-7:], dy2[:2], dy2[-7:] = float("nan"), float("inf"), float("nan"), -float("inf")
    w2[[e for e in range(E) if counts[e] == 0]] = float("nan")
    for f, a, b in ((ops.moe_grouped_matmul, (x, w), (x2, w2)), (ops.moe_grouped_matmul_dx, (dy, w), (dy2, w2)),
                    (ops.moe_grouped_matmul_dw, (dy, x), (dy2, x2))):
        assert torch.equal(f(*a, s), f(*b, s))
    x2 = x.clone()
    x2[7, 3] = float("nan")
    y, y2 = ops.moe_grouped_matmul(x, w, s), ops.moe_grouped_matmul(x2, w, s)
    keep = torch.arange(M, device=cuda) != 7
    assert bool(y2[7].isnan().all()) and torch.equal(y[keep], y2[keep])


@pytest.mark.parametrize("counts,N,K", TILED)
def test_tiled_captured_and_replayed(cuda, counts, N, K):
    ops, E, M = torch.ops.nanovllm, len(counts), sum(counts)
    x, w, dy = _rand(cuda, torch.float16, K, (M, K), (E, N, K), (M, N))
    assert tile_shape(M, N, K, E, 1)
    q, qs = ops.int8_quantize(w)
    starts = _starts(counts).to(cuda)

    def step():
        a = ops.int8_quantize(x)
        return (ops.moe_grouped_matmul(x, w, starts), ops.moe_grouped_matmul_dx(dy, w, starts), ops.moe_grouped_matmul_dw(dy, x, starts),
                ops.moe_grouped_matmul_int8(*a, q, qs, starts, torch.float32))

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i, c in enumerate((counts, counts[::-1], [M] + [0] * (E - 1), [0] * E)):
        a, b = _rand(cuda, torch.float16, 50 + i, (M, K), (M, N))
        x.copy_(a)
        dy.copy_(b)
        starts.copy_(_starts(c))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        for u, v in zip(out, want):
            assert torch.equal(u, v)


def test_tiled_on_two_streams(cuda):
    ops, sets = torch.ops.nanovllm, []
    for i, (counts, N, K) in enumerate(TILED):
        M, E = sum(counts), len(counts)
        x, w, dy = _rand(cuda, torch.bfloat16, 70 + i, (M, K), (E, N, K), (M, N))
        sets.append((x, w, dy, _starts(counts).to(cuda)))

    def step(x, w, dy, s):
        return ops.moe_grouped_matmul(x, w, s), ops.moe_grouped_matmul_dx(dy, w, s), ops.moe_grouped_matmul_dw(dy, x, s)

    want = [step(*a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for st, a in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(step(*a))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


# M, E, N, K: the few-rows kernel, sums that begin inside the row in tiles of 256 and of 128 columns, others
ORDER = [(700, 16, 520, 776), (4096, 128, 1536, 512), (1040, 16, 1544, 1280), (4100, 8, 2056, 1032)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("M,E,N,K", ORDER)
def test_results_follow_from_the_row_alone(cuda, dt, M, E, N, K):
    """At equal sizes a row's outputs do not depend, bit for bit, on how many rows its expert or others have, nor on where
    it lies; an expert's weight gradient does not depend on the others."""
    ops, e, most = torch.ops.nanovllm, E - 3, 300
    own, owndy, w, x, dy = _rand(cuda, DT[dt], M + E, (most, K), (most, N), (E, N, K), (M, K), (M, N))
    own[1], owndy[1] = own[0], owndy[0]   # two equal rows
    first = None
    for n, others in ((most, "even"), (most, "first"), (32, "even"), (128, "last"), (129, "even"), (20, "first"), (1, "none")):
        rest, c = M - n, [0] * E
        if others == "even":
            c = [rest // (E - 1)] * E
        elif others != "none":
            c[0 if others == "first" else E - 1] = rest
        c[e] = n
        s = _starts(c)
        a = int(s[e])
        x[a:a + n], dy[a:a + n] = own[:n], owndy[:n]
        s = s.to(cuda)
        y, dx = ops.moe_grouped_matmul(x, w, s)[a:a + n], ops.moe_grouped_matmul_dx(dy, w, s)[a:a + n]
        if first is None:
            first = y.clone(), dx.clone(), ops.moe_grouped_matmul_dw(dy, x, s)[e].clone()
            assert torch.equal(y[0], y[1]) and torch.equal(dx[0], dx[1])
        assert torch.equal(y, first[0][:n]) and torch.equal(dx, first[1][:n]), (n, others)
        if n == most:
            assert torch.equal(ops.moe_grouped_matmul_dw(dy, x, s)[e], first[2]), (n, others)


def _int8_exact(x, xs, w, ws, bias):
    """The sum, the scales' product and the bias in 64 bits (each operation off by at most 2^-53 of what it works on), rounded
    to fp32: half a step."""
    p = (x.double() @ w.double().t()) * (xs.double().unsqueeze(1) * ws.double())
    b = torch.zeros_like(ws, dtype=torch.float64) if bias is None else bias.double()
    return p + b, ref.round_bound(p + b, (p.abs() + b.abs()) * 2.0 ** -51, torch.float32)


@pytest.mark.parametrize("M,N,K", [(5, 300, 2048), (60, 1000, 4096), (200, 19001, 2048), (131, 20000, 1040), (1000, 2100, 1024),
                                   (128, 16001, 1040), (333, 1001, 8208), (2000, 6001, 272)])
def test_int8_fp32_outputs_rounded_once(cuda, M, N, K):
    """The few-rows kernel and each tile shape: 32-bit outputs have no rounding before the last."""
    x, xs, w, ws = _codes(cuda, N + K, (M, K), (N, K))
    bias = torch.randn(N, generator=torch.Generator(device="cuda").manual_seed(N), device=cuda)
    ops = torch.ops.nanovllm
    for b in (bias, None):
        assert ref.within(ops.int8_matmul(x, xs, w, ws, b, torch.float32), *_int8_exact(x, xs, w, ws, b)) <= 1.0
    s = _starts([M])
    y = ops.moe_grouped_matmul_int8(x, xs, w[None], ws[None], s.to(cuda), torch.float32)
    assert ref.within(y, *_int8_exact(x, xs, w, ws, None)) <= 1.0


@pytest.mark.parametrize("M,N,K", [(5, 300, 2048), (200, 19001, 2048), (131, 20000, 1040), (1000, 2100, 1024), (333, 1001, 8208),
                                   (2000, 6000, 272)])
def test_int8_scales_of_any_size(cuda, M, N, K):
    """A sum times one scale leaves the range of fp32, the output does not (every third channel alone, too); outputs below fp32's
    normal values; no sum gives 0 whatever the scales; a NaN scale gives NaN."""
    f = torch.ops.nanovllm.int8_matmul
    x, xs, w, ws = _codes(cuda, K, (M, K), (N, K))
    for a, b in ((1e-30, 1e38), (1e38, 1e-30), (1e-30, 1e-10), (1e-12, 1e-36), (1e-24, 1e-24)):
        xa, wb = xs * a, ws * b
        for third in (False, True):
            if third:
                wb = torch.where(torch.arange(N, device=cuda) % 3 == 0, wb, ws * 1e3)
                if a > 1:   # outputs of the others would leave the range themselves
                    wb[torch.arange(N, device=cuda) % 3 != 0] = b
            assert ref.within(f(x, xa, w, wb, None, torch.float32), *_int8_exact(x, xa, w, wb, None)) <= 1.0, (a, b)
            assert ref.within(f(x, xa, w, wb, None, torch.bfloat16), *ref.int8_rows(x, xa, w, wb, None, torch.bfloat16)) <= 1.0, (a, b)
    zero = torch.zeros_like(x)
    ws[1] = float("nan")
    for out in OUT:
        y = f(zero, xs * 1e35, w, ws * 1e35, None, out)
        assert bool(y[:, 1].isnan().all()) and not bool(y[:, 2:].any()) and not bool(y[:, 0].any())


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("cols", [2048, 2047])
def test_dequantized_values_bit_for_bit(cuda, out, cols):
    """code * scale in fp32, then rounded to the output's type, in every type: products of 31 bits that fp32 rounds to a tie of
    16 bits are among them (one in some thousands)."""
    q, s = _codes(cuda, cols, (4096, cols))
    want = (q.float() * s.unsqueeze(1)).to(out)
    assert torch.equal(torch.ops.nanovllm.int8_dequantize(q, s, out), want)
