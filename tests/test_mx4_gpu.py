"""Matrices in microscaled 4-bit numbers: the stored bytes against the definition, the products and the experts against 64 bits on the same
microscaled values, and the calls around them (graphs, streams, buffers that begin anywhere)."""
import pytest
import torch

import plain_mx4 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def normal(shape, seed, dtype=BF16, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


def quantised(w):
    from minfer_amd.kernels import ops
    codes, powers = (torch.full(s, 0xA5, dtype=torch.uint8, device=DEV) for s in ops.mx4_shapes(*w.shape))
    ops.mx4_quantise(w, codes, powers)
    return codes, powers


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(out, want, bound):
    off = (out.double() - want).abs()
    ok = (off <= bound) | (torch.isnan(want) & torch.isnan(out.double()))
    assert ok.all(), f"{int((~ok).sum())} of {ok.numel()} off, by up to {(off / bound)[~ok].max().item():.3g} of what they may"


# ------------------------------------------------------------------ quantising
@pytest.mark.parametrize("rows,k", [(1, 1), (16, 128), (17, 33), (128, 896), (5, 4095), (100, 520), (33, 1028)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantise_and_back(rows, k, dtype):
    from minfer_amd.kernels import ops
    w = normal((rows, k), rows + k, dtype, 0.02)
    codes, powers = quantised(w)
    want = plain.stored(w)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(powers.cpu(), want[1])
    held = plain.read(codes, powers, rows, k)
    for back in (BF16, F32):
        out = torch.full((rows, k), float("nan"), dtype=back, device=DEV)
        ops.mx4_dequantise(codes, powers, out)
        assert torch.equal(out.double(), held)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantise_every_kind_of_block(dtype):
    """Zeros, the smallest and the largest numbers, largest values on both sides of where the power moves on, every middle between two values,
    infinities and NaN."""
    from minfer_amd.kernels import ops
    top = torch.finfo(dtype).max
    first = [0.0, 2.0 ** -133, 2.0 ** -127, 2.0 ** -126, 2.0 ** -125, 1.75, 1.7578125, 7.0, 7.03125, 3.5, 1e30, top, float("inf"), -float("inf"), float("nan")]
    levels = [0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0]
    rows = []
    for i, v in enumerate(first):
        scale = abs(v) / 7.0 if 0 < abs(v) < 1e31 else 1.0 if abs(v) < 1 else 1e30
        row = [l * scale * (-1) ** (j + i) for j, l in enumerate(levels)] + [v] + [0.0] * 15
        rows.append(row + [1.0] * 7)                                       # and a short block behind it
    rows.append([x * 2.0 ** 20 for x in levels] + [-x * 2.0 ** 20 for x in levels] + [-0.0] * 7)
    w = torch.tensor(rows, dtype=torch.float64).to(dtype).to(DEV)
    codes, powers = quantised(w)
    want = plain.stored(w)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(powers.cpu(), want[1])
    held = plain.read(codes, powers, *w.shape)
    out = torch.empty(w.shape, dtype=F32, device=DEV)
    ops.mx4_dequantise(codes, powers, out)
    assert torch.equal(torch.isnan(out), torch.isnan(held)) and torch.isnan(held).any()
    assert torch.equal(out.nan_to_num(0.0).double(), held.to(F32).nan_to_num(0.0).double())
    # half a step: 1/2 of a block's power, 1 above 2, 2 above 4
    finite = torch.isfinite(w.double()).all(1)
    power = plain.power_of_two(plain.nearest(w, plain.E2M1)[1]).repeat_interleave(32, 1)[:, :w.shape[1]]
    ratio = w.double().abs() / power
    step = torch.where(ratio < 2, 0.5, torch.where(ratio < 4, 1.0, 2.0))
    assert ((held - w.double()).abs() <= step / 2 * power)[finite].all()


# ------------------------------------------------------------------ products
SIZES = [(16, 32), (896, 896), (130, 1000), (1100, 2500), (48, 128), (300, 5000), (2048, 640)]


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 129, 300])
@pytest.mark.parametrize("n,k", SIZES)
def test_linear(m, n, k):
    from minfer_amd.kernels import ops
    for number, (dtype, out_dtype, with_bias, add) in enumerate([(BF16, F32, False, False), (F32, BF16, True, False), (BF16, F32, True, True)]):
        x = normal((m, k), m + n + number, dtype)
        codes, powers = quantised(normal((n, k), n + k, std=0.05))
        bias = normal((n,), 7, F32) if with_bias else None
        before = normal((m, n), 8, F32)
        out = before.to(out_dtype).clone() if add else torch.full((m, n), float("nan"), dtype=out_dtype, device=DEV)
        ops.mx4_linear(x, codes, powers, bias, out, accumulate=add)
        want, size = plain.product(x, plain.read(codes, powers, n, k))
        bound = plain.sum_error(k, size + (bias.double().abs() if with_bias else 0) + (before.double().abs() if add else 0))
        want = want + (bias.double() if with_bias else 0) + (before.double() if add else 0)
        within(out, want, bound + half_step(out_dtype) * (want.abs() + bound) + 1e-37)


@pytest.mark.parametrize("m,n,k", [(2048, 4608, 512), (700, 3584, 2048), (520, 896, 4864), (4096, 1024, 256), (257, 8208, 130), (100, 512, 18944)])
def test_linear_of_prompts(m, n, k):
    from minfer_amd.kernels import ops
    x, bias = normal((m, k), m + n), normal((n,), 7, F32)
    codes, powers = quantised(normal((n, k), n + k, std=0.05))
    out = torch.full((m, n), float("nan"), device=DEV)
    ops.mx4_linear(x, codes, powers, bias, out)
    want, size = plain.product(x, plain.read(codes, powers, n, k))
    bound = plain.sum_error(k, size + bias.double().abs())
    within(out, want + bias.double(), bound + half_step(F32) * (want.abs() + bound) + 1e-37)


@pytest.mark.parametrize("m", [1, 16, 31, 64, 70, 260, 600])
@pytest.mark.parametrize("f,k", [(16, 128), (300, 700), (1000, 96), (37, 4100), (4864, 896)])
def test_linear_swiglu(m, f, k):
    from minfer_amd.kernels import ops
    x = normal((m, k), m + f, F32 if m == 31 else BF16)
    gate, up = quantised(normal((f, k), 1, std=0.05)), quantised(normal((f, k), 2, std=0.05))
    out = torch.full((m, f), float("nan"), dtype=BF16, device=DEV)
    ops.mx4_linear_swiglu(x, ops.mx4_pairs(gate[0], up[0]), ops.mx4_pairs(gate[1], up[1]), out)
    (g, g_size), (u, u_size) = (plain.product(x, plain.read(*t, f, k)) for t in (gate, up))
    dg, du = plain.sum_error(k, g_size), plain.sum_error(k, u_size)
    want = plain.silu(g) * u
    # |silu'| is below 1.1 and |silu(g)| below |g|; silu itself: 2^x and a reciprocal of 32 bits, the argument's rounding times its size
    bound = 1.1 * dg * (u.abs() + du) + g.abs() * du + (g.abs() + 16) * 2.0 ** -22 * want.abs()
    within(out, want, bound + half_step(BF16) * (want.abs() + bound) + 1e-37)


# (kernel, whether K is cut over blocks, m, n, k): each tile kernel at sizes where the plan takes it, with tiles that end outside
TILED = [(2, False, 6404, 4408, 5899), (3, False, 396, 8626, 64), (3, True, 1625, 2795, 15905), (4, False, 2778, 720, 84), (4, True, 720, 1508, 8730),
         (5, False, 46, 65, 67), (5, True, 66, 72, 3114)]
TILED_GATES = [(2, False, 3484, 4102, 6683), (3, False, 772, 2662, 66), (3, True, 1297, 1535, 17507), (4, False, 196, 6430, 64),
               (4, True, 257, 804, 12727), (5, False, 70, 333, 200), (5, True, 42, 70, 3383)]


def planned(kernel, cut, m, n, k, epi):
    from minfer_amd.kernels import ops
    if ops.cu_count() == 256:
        form, parts, _, _ = ops._mx4_plan(m, n, k, epi, 1, 256)
        assert (form, parts > 1) == (kernel, cut)


@pytest.mark.parametrize("kernel,cut,m,n,k", TILED)
def test_linear_in_every_tile_kernel(kernel, cut, m, n, k):
    from minfer_amd.kernels import ops
    planned(kernel, cut, m, n, k, ops.EPI_ACC_F32)
    x, bias, before = normal((m, k), m + n), normal((n,), 7, F32), normal((m, n), 8, F32)
    codes, powers = quantised(normal((n, k), n + k, std=0.05))
    want, size = plain.product(x, plain.read(codes, powers, n, k))
    for add, out_dtype in ((True, F32), (False, BF16)):
        out = before.clone() if add else torch.full((m, n), float("nan"), dtype=out_dtype, device=DEV)
        ops.mx4_linear(x, codes, powers, bias, out, accumulate=add)
        bound = plain.sum_error(k, size + bias.double().abs() + (before.double().abs() if add else 0))
        whole = want + bias.double() + (before.double() if add else 0)
        within(out, whole, bound + half_step(out_dtype) * (whole.abs() + bound) + 1e-37)


@pytest.mark.parametrize("kernel,cut,m,f,k", TILED_GATES)
def test_linear_swiglu_in_every_tile_kernel(kernel, cut, m, f, k):
    from minfer_amd.kernels import ops
    planned(kernel, cut, m, f, k, ops.EPI_SWIGLU)
    x = normal((m, k), m + f)
    gate, up = quantised(normal((f, k), 1, std=0.05)), quantised(normal((f, k), 2, std=0.05))
    out = torch.full((m, f), float("nan"), dtype=BF16, device=DEV)
    ops.mx4_linear_swiglu(x, ops.mx4_pairs(gate[0], up[0]), ops.mx4_pairs(gate[1], up[1]), out)
    (g, g_size), (u, u_size) = (plain.product(x, plain.read(*t, f, k)) for t in (gate, up))
    dg, du = plain.sum_error(k, g_size), plain.sum_error(k, u_size)
    want = plain.silu(g) * u
    bound = 1.1 * dg * (u.abs() + du) + g.abs() * du + (g.abs() + 16) * 2.0 ** -22 * want.abs()        # (as in test_linear_swiglu)
    within(out, want, bound + half_step(BF16) * (want.abs() + bound) + 1e-37)


@pytest.mark.parametrize("m", [7, 48, 130])
def test_linear_swiglu_clamped(m):
    from minfer_amd.kernels import ops
    f, k, limit = 90, 260, 0.7
    x = normal((m, k), m)
    gate, up = quantised(normal((f, k), 1, std=0.05)), quantised(normal((f, k), 2, std=0.05))
    out = torch.full((m, f), float("nan"), dtype=BF16, device=DEV)
    ops.mx4_linear_swiglu(x, ops.mx4_pairs(gate[0], up[0]), ops.mx4_pairs(gate[1], up[1]), out, limit=limit)
    (g, g_size), (u, u_size) = (plain.product(x, plain.read(*t, f, k)) for t in (gate, up))
    want = plain.act(g, u, limit, 0)
    # the gate's slope is below 1.2 and itself below the limit, u + 1 at most limit + 1
    bound = 1.2 * (limit + 1) * plain.sum_error(k, g_size) + limit * plain.sum_error(k, u_size) + (g.abs() + 16) * 2.0 ** -22 * (limit + 1)
    within(out, want, bound + half_step(BF16) * (want.abs() + bound))


def test_rows_apart():
    """An infinity or a NaN in a row of x makes that row NaN and no other; a NaN block of the matrix makes its output NaN in every row."""
    from minfer_amd.kernels import ops
    for m in (5, 40, 100):
        x = normal((m, 300), m)
        x[1, 7], x[3, 299] = float("inf"), float("nan")
        w = normal((70, 300), 3, std=0.05)
        w[66, 100] = float("nan")
        codes, powers = quantised(w)
        out = torch.empty((m, 70), device=DEV)
        ops.mx4_linear(x, codes, powers, None, out)
        bad = torch.zeros((m, 70), dtype=torch.bool, device=DEV)
        bad[1], bad[3], bad[:, 66] = True, True, True
        assert torch.equal(torch.isnan(out), bad)
        clean = x.clone()
        clean[1, 7] = clean[3, 299] = 0
        again = torch.empty_like(out)
        ops.mx4_linear(clean, codes, powers, None, again)
        assert torch.equal(out[~bad], again[~bad])


@pytest.mark.parametrize("scale_x,scale_w", [(1e-30, 1e-5), (1e25, 1e10), (2.0 ** -126, 2.0 ** 100), (0.0, 1.0)])
def test_far_powers(scale_x, scale_w):
    """Blocks near both ends of the powers, whose products are ordinary numbers, or too small for one; rows of zeros."""
    from minfer_amd.kernels import ops
    for m in (3, 70):
        x, w = (normal((m, 256), m, F32) * scale_x), normal((48, 256), 5, F32) * scale_w
        codes, powers = quantised(w)
        out = torch.full((m, 48), float("nan"), device=DEV)
        ops.mx4_linear(x, codes, powers, None, out)
        want, size = plain.product(x, plain.read(codes, powers, 48, 256))
        # (a product below 2^-126 may be taken as zero)
        within(out, want, plain.sum_error(256, size) + half_step(F32) * want.abs() + 256 * 2.0 ** -126)


def misaligned(t):
    base = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    base[1:] = t.flatten()
    return base[1:].view(t.shape)


@pytest.mark.parametrize("m", [3, 40, 90])
def test_operands_that_begin_anywhere(m):
    """x and out off 16 bytes, bias off 16; the bytes around out stay."""
    from minfer_amd.kernels import ops
    n, k = 96, 256
    x, bias = normal((m, k), m), normal((n,), 1, F32)
    codes, powers = quantised(normal((n, k), 2, std=0.05))
    for dtype in (F32, BF16):
        want = torch.empty((m, n), dtype=dtype, device=DEV)
        ops.mx4_linear(x, codes, powers, bias, want)
        around = torch.full((m * n + 129,), 3.0, dtype=dtype, device=DEV)
        out = around[65:65 + m * n].view(m, n)
        ops.mx4_linear(misaligned(x), codes, powers, misaligned(bias), out)
        assert torch.equal(out, want)
        assert (around[:65] == 3).all() and (around[65 + m * n:] == 3).all()


def guarded(shape, dtype, fill):
    """A tensor of this shape in the middle of a larger one full of `fill`, and a check that nothing around it changed."""
    n = torch.Size(shape).numel()
    base = torch.full((n + 2 * 4096,), fill, dtype=dtype, device=DEV)
    return base[4096:4096 + n].view(shape), lambda: bool((base[:4096] == fill).all() and (base[4096 + n:] == fill).all())


@pytest.mark.parametrize("m", [1, 5, 8, 13, 16, 19, 37, 64, 75, 200, 513])
@pytest.mark.parametrize("n,k", [(896, 896), (130, 1000), (37, 4097), (1003, 70)])
def test_nothing_outside_is_written(m, n, k):
    from minfer_amd.kernels import ops
    w = normal((n, k), 3, std=0.05)
    codes, codes_kept = guarded(ops.mx4_shapes(n, k)[0], torch.uint8, 0x5A)
    powers, powers_kept = guarded(ops.mx4_shapes(n, k)[1], torch.uint8, 0x5A)
    ops.mx4_quantise(w, codes, powers)
    back, back_kept = guarded((n, k), BF16, -7.0)
    ops.mx4_dequantise(codes, powers, back)
    assert codes_kept() and powers_kept() and back_kept() and (back != -7.0).any()
    x = normal((m, k), 4)
    both = ops.mx4_pairs(codes, codes), ops.mx4_pairs(powers, powers)
    for dtype, add in ((F32, False), (F32, True), (BF16, False)):
        out, kept = guarded((m, n), dtype, -7.0)
        ops.mx4_linear(x, codes, powers, None, out, accumulate=add)
        assert kept() and (out != -7.0).float().mean() > 0.99
    out, kept = guarded((m, n), BF16, -7.0)
    ops.mx4_linear_swiglu(x, *both, out)
    assert kept() and (out != -7.0).all()
    if m <= 16:
        down = quantised(normal((n, n), 5, std=0.05))
        experts_ = [t[None].repeat(3, *[1] * t.dim()) for t in (*both, *down)]
        chosen = torch.tensor([[i % 3, 2] for i in range(m)], dtype=torch.int32, device=DEV)
        out, kept = guarded((m, n), BF16, -7.0)
        ops.mx4_moe_sparse(x, *experts_, chosen, torch.ones((m, 2), device=DEV), out, n, act=1, accumulate=False)
        assert kept() and (out != -7.0).float().mean() > 0.99


def test_no_rows():
    from minfer_amd.kernels import ops
    codes, powers = quantised(normal((32, 64), 1))
    ops.mx4_linear(torch.empty((0, 64), dtype=BF16, device=DEV), codes, powers, None, torch.empty((0, 32), device=DEV))


def test_codes_past_four_gigabytes():
    """The last rows of a matrix whose codes pass 2^32 bytes."""
    from minfer_amd.kernels import ops
    k, rows = 8192, (1 << 20) + 40
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("not enough memory")
    shapes = ops.mx4_shapes(rows, k)
    codes = torch.randint(0, 256, shapes[0], dtype=torch.uint8, device=DEV)
    powers = torch.randint(120, 130, shapes[1], dtype=torch.uint8, device=DEV)
    assert codes.numel() > 1 << 32
    tail = plain.read(codes[-3:], powers[-3:], 40, k)                      # (rows end inside the last tile)
    for m in (2, 20, 70):
        x = normal((m, k), m)
        out = torch.empty((m, rows), device=DEV)
        ops.mx4_linear(x, codes, powers, None, out)
        want, size = plain.product(x, tail)
        within(out[:, -40:], want, plain.sum_error(k, size) + half_step(F32) * want.abs())
        del out


# ------------------------------------------------------------------ experts
def experts(e, f, k, seed, n=None):
    """(gate_up, powers, down, powers) as the layer takes them, and the values of gate, up, down in 64 bits."""
    from minfer_amd.kernels import ops
    n = k if n is None else n
    made = [[quantised(normal(s, seed + 3 * i + j, std=0.05)) for i in range(e)] for j, s in enumerate(((f, k), (f, k), (n, f)))]
    gate, up, down = ([torch.stack([t[q] for t in made[j]]) for q in (0, 1)] for j in range(3))
    held = [plain.read(*t, *s) for t, s in ((gate, (f, k)), (up, (f, k)), (down, (n, f)))]
    return (ops.mx4_pairs(gate[0], up[0]), ops.mx4_pairs(gate[1], up[1]), *down), held


def experts_plain(x, held, chosen, weights, limit, kind):
    """(outputs, what they may be off): a value of y whose rounding goes the other way within the sums' error moves its E2M3 value by a step."""
    gate, up, down = held
    out = torch.zeros((x.shape[0], down.shape[1]), dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(out)
    k, f = gate.shape[2], gate.shape[1]
    for t in range(x.shape[0]):
        for j, e in enumerate(chosen[t].tolist()):
            if not 0 <= e < gate.shape[0]:
                continue
            (g, gs), (u, us) = plain.product(x[t:t + 1], gate[e]), plain.product(x[t:t + 1], up[e])
            dg, du = plain.sum_error(k, gs), plain.sum_error(k, us)
            y = plain.act(g, u, limit, kind)
            # slopes: of the gates below 1.2, of their products with u; the clamped form adds 1 to u
            dy = 1.2 * dg * (u.abs() + du + 1) + (g.abs() + 1) * du + (g.abs() + 16) * 2.0 ** -22 * y.abs()
            near, low, high = (plain.rows6((y + s).to(torch.bfloat16)) for s in (0.0, -torch.sign(y) * dy, torch.sign(y) * dy))
            moved = torch.maximum((high - near).abs(), (low - near).abs())
            w = weights[t, j].double()
            z, size = near @ down[e].T, (near.abs() + moved) @ down[e].abs().T
            out[t] += (w * z)[0]
            bound[t] += (w.abs() * (moved @ down[e].abs().T + plain.sum_error(f, size) + 2.0 ** -23 * size))[0]
    return out, bound


@pytest.mark.parametrize("tokens,top,e,f,k", [(1, 1, 1, 16, 32), (1, 4, 32, 192, 256), (3, 2, 4, 100, 130), (8, 2, 8, 512, 256), (16, 8, 16, 64, 300),
                                              (16, 1, 3, 260, 1000), (2, 64, 64, 48, 64), (5, 3, 3, 130, 777)])
@pytest.mark.parametrize("kind,limit", [(1, 0.0), (0, 0.7)])
def test_experts(tokens, top, e, f, k, kind, limit):
    from minfer_amd.kernels import ops
    layer, held = experts(e, f, k, 10 * e)
    gen = torch.Generator().manual_seed(tokens + e)
    chosen = torch.rand((tokens, e), generator=gen).argsort(-1)[:, :top].to(torch.int32).contiguous().to(DEV)
    weights = torch.softmax(torch.randn((tokens, top), generator=gen), -1).to(DEV)
    for dtype, out_dtype, add in ((BF16, F32, True), (F32, F32, False), (BF16, BF16, False)):
        x = normal((tokens, k), tokens + k, dtype)
        want, bound = experts_plain(x, held, chosen, weights, limit, kind)
        before = normal((tokens, k), 5, F32)
        out = before.clone() if add else torch.full((tokens, k), float("nan"), dtype=out_dtype, device=DEV)
        ops.mx4_moe_sparse(x, *layer, chosen, weights, out, f, limit, kind, accumulate=add)
        if add:
            want = want + before.double()
        within(out, want, bound + (2.0 ** -23 + half_step(out_dtype)) * (want.abs() + bound) + 1e-37)


def test_experts_odd_choices():
    """The same expert twice for one token, choices that name none (below 0 and past the last), a token without any, outputs of another width."""
    from minfer_amd.kernels import ops
    e, f, k, n = 4, 96, 160, 80
    layer, held = experts(e, f, k, 3, n)
    chosen = torch.tensor([[1, 1, 2], [-1, 4, 7], [3, -5, 3], [0, 1, 2]], dtype=torch.int32, device=DEV)
    weights = torch.rand((4, 3), generator=torch.Generator().manual_seed(1)).to(DEV)
    x = normal((4, k), 9)
    want, bound = experts_plain(x, held, chosen, weights, 0.0, 1)
    out = torch.full((4, n), float("nan"), device=DEV)
    ops.mx4_moe_sparse(x, *layer, chosen, weights, out, f, act=1, accumulate=False)
    within(out, want, bound + half_step(F32) * want.abs() + 1e-37)
    assert (out[1] == 0).all()


@pytest.mark.parametrize("tokens", [3, 7, 12])
def test_experts_keep_tokens_apart(tokens):
    """A token with an infinity is NaN; the others are what they are without it, whoever shares their experts."""
    from minfer_amd.kernels import ops
    e, f, k = 5, 96, 160
    layer, _ = experts(e, f, k, 8)
    gen = torch.Generator().manual_seed(tokens)
    chosen = torch.rand((tokens, e), generator=gen).argsort(-1)[:, :2].to(torch.int32).contiguous().to(DEV)
    weights = torch.rand((tokens, 2), generator=gen).to(DEV)
    x = normal((tokens, k), 4)
    bad = x.clone()
    bad[1, 5] = float("inf")
    outs = []
    for rows in (x, bad):
        outs.append(torch.full((tokens, k), float("nan"), device=DEV))
        ops.mx4_moe_sparse(rows, *layer, chosen, weights, outs[-1], f, act=1, accumulate=False)
    assert torch.isnan(outs[1][1]).all() and torch.isfinite(outs[0]).all()
    others = [t for t in range(tokens) if t != 1]
    assert torch.equal(outs[0][others], outs[1][others])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_experts_that_hand_on(dtype):
    from minfer_amd.kernels import ops
    e, f, k = 3, 64, 96
    layer, held = experts(e, f, k, 4)
    chosen = torch.tensor([[0, 3], [4, 3], [2, 1]], dtype=torch.int32, device=DEV)
    weights = torch.rand((3, 2), generator=torch.Generator().manual_seed(2)).to(DEV)
    x = normal((3, k), 6, dtype)
    want, bound = experts_plain(x, held, chosen, weights, 0.0, 1)
    want += ((chosen >= e) * weights.double()).sum(1, keepdim=True) * x.double()
    out = torch.zeros((3, k), device=DEV)
    ops.mx4_moe_sparse(x, *layer, chosen, weights, out, f, act=1, hands_on=True)
    within(out, want, bound + 4 * half_step(F32) * (want.abs() + x.double().abs()) + 1e-37)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens", [2, 6, 16])
def test_experts_of_rows_that_begin_anywhere(tokens, dtype):
    """x, outputs and the rows handed on at odd addresses: the same bits as from aligned ones."""
    from minfer_amd.kernels import ops
    e, f, k = 4, 96, 168
    layer, _ = experts(e, f, k, 5)
    gen = torch.Generator().manual_seed(tokens)
    chosen = torch.randint(0, e + 2, (tokens, 3), generator=gen).to(torch.int32).to(DEV)
    weights = torch.rand((tokens, 3), generator=gen).to(DEV)
    x = normal((tokens, k), 6, dtype)
    outs = []
    for rows, out in ((x, torch.zeros((tokens, k), device=DEV)), (misaligned(x), misaligned(torch.zeros((tokens, k), device=DEV)))):
        ops.mx4_moe_sparse(rows, *layer, chosen, weights, out, f, act=1, hands_on=True)
        outs.append(out)
    assert outs[0].any(1).all() and torch.equal(*outs)


# ------------------------------------------------------------------ as they are used
def feed_forward(x, weights, h):
    """down(silu(gate x) up x), added to h."""
    from minfer_amd.kernels import ops
    y = torch.empty((x.shape[0], weights["f"]), dtype=BF16, device=DEV)
    ops.mx4_linear_swiglu(x, *weights["gate_up"], y)
    ops.mx4_linear(y, *weights["down"], None, h, accumulate=True)
    return y


def feed_forward_weights(f, k, seed):
    from minfer_amd.kernels import ops
    gate, up, down = (quantised(normal(s, seed + i, std=0.05)) for i, s in enumerate(((f, k), (f, k), (k, f))))
    return dict(f=f, gate_up=(ops.mx4_pairs(gate[0], up[0]), ops.mx4_pairs(gate[1], up[1])), down=down)


@pytest.mark.parametrize("m", [1, 12, 50, 200])
def test_a_feed_forward(m):
    """Quantised once, then one product behind the other: each against 64 bits on what it was given."""
    f, k = 300, 256
    weights = feed_forward_weights(f, k, 1)
    x, h = normal((m, k), m), normal((m, k), 2, F32)
    out = h.clone()
    y = feed_forward(x, weights, out)
    want, size = plain.product(y, plain.read(*weights["down"], k, f))
    bound = plain.sum_error(f, size + h.double().abs())
    within(out, want + h.double(), bound + half_step(F32) * (want.abs() + bound))


@pytest.mark.parametrize("m", [4, 40, 150])
def test_captured_and_replayed(m):
    """Two graphs and eager calls in turn, on inputs that change between the replays: the same bits."""
    f, k = 512, 384
    weights = feed_forward_weights(f, k, 3)
    layer, _ = experts(4, 64, k, 5)
    chosen = torch.tensor([[0, 2]] * min(m, 16), dtype=torch.int32, device=DEV)
    share = torch.full((min(m, 16), 2), 0.5, device=DEV)
    x, h = torch.zeros((m, k), dtype=BF16, device=DEV), torch.zeros((m, k), device=DEV)

    def work():
        from minfer_amd.kernels import ops
        feed_forward(x, weights, h)
        ops.mx4_moe_sparse(x[:16], *layer, chosen, share, h[:16], 64, act=1)
    work()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            work()
        graphs.append(graph)
    for i in range(6):
        x.copy_(normal((m, k), 100 + i))
        h.zero_()
        work()
        want = h.clone()
        h.zero_()
        graphs[i % 2].replay()
        assert torch.equal(h, want)
        torch.cuda.synchronize()


def test_two_streams_at_once():
    """Calls on two streams share nothing."""
    f, k, m = 1024, 2048, 300
    weights = feed_forward_weights(f, k, 7)
    xs = [normal((m, k), i) for i in range(2)]
    want = []
    for x in xs:
        h = torch.zeros((m, k), device=DEV)
        feed_forward(x, weights, h)
        want.append(h)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [torch.zeros((m, k), device=DEV) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, x, h in zip(streams, xs, got):
            with torch.cuda.stream(s):
                h.zero_()
                feed_forward(x, weights, h)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------ refusals
def test_refusals():
    from minfer_amd.kernels import ops
    codes, powers = quantised(normal((64, 256), 1))
    x, out = normal((3, 256), 2), torch.empty((3, 64), device=DEV)

    def refused(call, *parts):
        with pytest.raises(ops.KernelError) as e:
            call()
        assert all(p in str(e.value) for p in parts), str(e.value)
    refused(lambda: ops.mx4_linear(x.half(), codes, powers, None, out), "mx4_linear.x", "float16")
    refused(lambda: ops.mx4_linear(x[:, ::2], codes, powers, None, out), "contiguous")
    refused(lambda: ops.mx4_linear(x, codes[:2], powers, None, out), "mx4_linear.codes", "shape")
    refused(lambda: ops.mx4_linear(x, codes, powers[:, :, :32].contiguous(), None, out), "mx4_linear.powers")
    refused(lambda: ops.mx4_linear(x[:, :128].contiguous(), codes, powers, None, out), "mx4_linear.codes")
    refused(lambda: ops.mx4_linear(x, codes, powers, torch.zeros(63, device=DEV), out), "mx4_linear.bias")
    refused(lambda: ops.mx4_linear(x, codes, powers, None, out[:2]), "mx4_linear")
    refused(lambda: ops.mx4_linear(x, codes, powers, None, out.to(BF16), accumulate=True), "accumulation")
    refused(lambda: ops.mx4_linear(x.cpu(), codes, powers, None, out), "GPU")
    refused(lambda: ops.mx4_linear(x, misaligned(codes), powers, None, out), "16 bytes")
    refused(lambda: ops.mx4_linear_swiglu(x, codes, powers, torch.empty((3, 64), dtype=BF16, device=DEV)), "mx4_linear_swiglu.codes")
    refused(lambda: ops.mx4_linear_swiglu(x, codes, powers, out), "bfloat16")
    refused(lambda: ops.mx4_quantise(normal((64, 255), 1), codes, powers.view(torch.int8)), "mx4_quantise.powers")
    refused(lambda: ops.mx4_quantise(normal((2, 64, 256), 1), codes, powers), "matrix")
    refused(lambda: ops.mx4_quantise(torch.empty((0, 256), device=DEV), codes, powers), "sizes")
    refused(lambda: ops.mx4_dequantise(codes, powers, torch.empty((65, 256), device=DEV)), "mx4_dequantise.codes")
    layer, _ = experts(2, 32, 64, 1)
    rows, two = normal((3, 64), 1), torch.zeros((3, 2), dtype=torch.int32, device=DEV)
    share, h = torch.ones((3, 2), device=DEV), torch.zeros((3, 64), device=DEV)
    refused(lambda: ops.mx4_moe_sparse(rows, *layer, two.long(), share, h, 32), "mx4_moe_sparse.chosen")
    refused(lambda: ops.mx4_moe_sparse(rows, *layer, two, share, h, 48), "mx4_moe_sparse.gate_up")
    refused(lambda: ops.mx4_moe_sparse(rows, *layer, two, share, h.to(BF16), 32), "accumulation")
    refused(lambda: ops.mx4_moe_sparse(rows, *layer, two, share, h, 32, act=2), "activation")
    many = normal((17, 64), 1), torch.zeros((17, 1), dtype=torch.int32, device=DEV), torch.ones((17, 1), device=DEV), torch.zeros((17, 64), device=DEV)
    refused(lambda: ops.mx4_moe_sparse(many[0], *layer, many[1], many[2], many[3], 32), "17 tokens")
    torch.cuda.synchronize()
