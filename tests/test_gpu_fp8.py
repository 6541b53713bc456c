"""The block-scaled FP8 products and the group-limited router against plain
64-bit forms of their definitions, on the GPU.

Tolerances, from the arithmetic (u32 = 2^-24, bf16 half step 2^-8):

- Quantized values and scales are defined with 32-bit roundings at fixed
  places: compared bit for bit.
- linear: products of E4M3 values are exact; a sum of K of them (and the K / 128
  block sums times two scales) in fp32 is off by at most (K + 4) * 2^-23 of the
  sum S of magnitudes (2^-23: the tensor core may cut instead of round); the
  output is rounded once: |err| <= 2^-8 |y| + (K + 4) 2^-23 S (1 + 2^-8).
- feed-forward: hidden values differ from the 64-bit ones by a relative d of
  about 2^-23 sqrt(K) S / |h|, at most 1e-4 for these sizes. A value moves by one E4M3 step (at
  most 2^-3 of it) where a rounding border lies in between, which happens for
  a share of at most 2 d / 2^-4 of them, so the hidden rows' relative L2 is
  off by at most sqrt(32 d) 2^-3 = 7e-3; of a routed sum the rows are rounded
  to bf16 first and the sum after that: 2^-8 each (the mean square of a
  rounding error is a third of the largest: 2^-8 / sqrt(3) each in L2). In all
  sqrt(7e-3^2 + 2 * (2^-8)^2 / 3) < 1e-2, the layer's tolerance.
"""

from __future__ import annotations

import math

import pytest
import torch
from conftest import pkg

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
F8 = torch.float8_e4m3fn
DEV = "cuda"


@pytest.fixture(scope="module")
def P():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    p = pkg()
    p.capi.load()
    return p


@pytest.fixture(autouse=True)
def no_device_error(P):
    yield
    assert P.capi.device_error(0) == 0


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def blocks(x, rows):
    """[.., R, C] -> [.., ceil(R / rows), rows, ceil(C / 128), 128], zero-padded."""
    r, c = x.shape[-2:]
    x = torch.nn.functional.pad(x, (0, -c % 128, 0, -r % rows))
    return x.unflatten(-1, (-1, 128)).unflatten(-3, (-1, rows))


def unblock(b, r, c):
    return b.flatten(-4, -3).flatten(-2, -1)[..., :r, :c]


def quantized(x, rows=1):
    """(codes as fp32, scales) of fp32 x by the definition: per block of `rows`
    x 128, both quotients and the product rounded to 32 bits."""
    b = blocks(x, rows)
    a = b.abs().amax(dim=(-3, -1), keepdim=True).clamp(min=1e-12)
    most = torch.full_like(a, 448.0)
    codes = unblock((b * (most / a)).to(F8).float(), *x.shape[-2:])
    return codes, (a / most)[..., 0, :, 0]


def values(codes, scale, rows=1):
    """The 64-bit values of codes and block scales."""
    b = blocks(codes.double(), rows)
    return unblock(b * scale.double()[..., :, None, :, None], *codes.shape[-2:])


def rows64(x):
    return values(*quantized(x.float()))


def weight(g, *shape):
    """E4M3 weight with scales that differ from block to block by up to 2^6."""
    w = torch.randn(*shape, generator=g) * 0.02
    n, k = shape[-2:]
    lift = 2.0 ** torch.randint(-3, 4, shape[:-2] + (-(-n // 128), -(-k // 128)), generator=g).float()
    w = unblock(blocks(w, 128) * lift[..., :, None, :, None], n, k)
    codes, scale = quantized(w, 128)
    return codes.to(F8).to(DEV).contiguous(), scale.to(DEV).contiguous()


def w64(q, scale):
    return values(q.float(), scale, 128)


def swiglu64(x, gate_up, down):
    g, u = (x @ gate_up.mT).chunk(2, dim=-1)
    h = g / (1 + torch.exp(-g)) * u
    a = blocks(h, 1).abs().amax(dim=(-3, -1), keepdim=True).clamp(min=1e-12)
    r, s = (448.0 / a).float().double(), (a / 448.0).float().double()
    hq = unblock((blocks(h, 1) * r).to(F8).double() * s, *h.shape[-2:])
    return hq @ down.mT


def experts64(x, top, gate, gu, down, scaling):
    y = torch.zeros_like(x)
    for e in range(gu.shape[0]):
        t, s = torch.nonzero(top == e, as_tuple=True)
        if t.numel():
            y.index_add_(0, t, swiglu64(x[t], gu[e], down[e]) * (gate[t, s].double() * scaling)[:, None])
    return y


def rel(a, b):
    return float((a.double() - b).norm() / b.norm().clamp(min=1e-300))


def same_bits(a, b):
    return a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# -- quantization ------------------------------------------------------------

@pytest.mark.parametrize("r,k", [(1, 16), (1, 128), (3, 144), (33, 1040), (257, 2048), (1000, 384)])
def test_quantize_is_bit_exact(P, r, k):
    g = gen(r + k)
    x = randn(g, r, k) * torch.exp(2 * randn(g, 1, k, dtype=torch.float32)).to(BF16)
    x[0] = 0
    x[-1, : k // 2] = 1e-20
    q, scale = P.ops.fp8_quantize(x)
    codes, want = quantized(x.float())
    assert q.shape == x.shape and scale.shape == (r, -(-k // 128))
    assert torch.equal(q.float(), codes) and torch.equal(scale, want)


def test_quantize_rows_with_a_pitch_and_none(P):
    g = gen(5)
    wide = randn(g, 37, 512)
    x = wide[:, 128:384]
    q, scale = P.ops.fp8_quantize(x)
    codes, want = quantized(x.float())
    assert torch.equal(q.float(), codes) and torch.equal(scale, want)
    q, scale = P.ops.fp8_quantize(wide[:0])
    assert q.shape == (0, 512) and scale.shape == (0, 4)


@pytest.mark.parametrize("shape", [(128, 128), (144, 77), (3, 256, 300), (2, 1040, 128)])
def test_pack_weights_is_bit_exact(P, shape):
    w = randn(gen(sum(shape)), *shape, scale=0.02)
    q, scale = P.ops.fp8_pack_weights(w)
    codes, want = quantized(w.float().mT, 128)
    assert torch.equal(q.float(), codes) and torch.equal(scale, want)


# -- linear --------------------------------------------------------------------

def check_linear(y, x, q, s):
    xv, wv = rows64(x), w64(q, s)
    want = xv @ wv.T
    mag = xv.abs() @ wv.abs().T
    tol = 2.0**-8 * want.abs() + (x.shape[-1] + 4) * 2.0**-23 * mag * (1 + 2.0**-8)
    over = (y.double() - want).abs() - tol
    assert y.dtype == BF16 and not (over > 0).any(), float((over / tol).max())


LINEAR = [(1, 1, 16), (1, 256, 128), (1, 4096, 2048), (2, 129, 272), (3, 7, 48), (5, 1000, 400), (8, 512, 128),
          (9, 640, 1024), (16, 1001, 1040), (17, 264, 512), (33, 2048, 256), (64, 136, 384), (77, 1001, 1040),
          (128, 128, 128), (129, 257, 144), (255, 384, 1152), (300, 512, 2048), (513, 1030, 272), (1000, 4096, 512),
          (2100, 2312, 784), (1100, 2501, 272), (8, 40, 24576), (1, 33, 32768)]


@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear(P, m, n, k):
    g = gen(m * 7 + n + k)
    q, s = weight(g, n, k)
    x = randn(g, m, k)
    y = P.ops.fp8_linear(x, q, s)
    check_linear(y, x, q, s)
    assert same_bits(y, P.ops.fp8_linear(x, q, s))


@pytest.mark.parametrize("m", [9, 17, 31, 32, 33])
@pytest.mark.parametrize("n,k", [(9504, 128), (9728, 272), (9760, 1040), (9496, 256), (10001, 144)])
def test_linear_few_rows_of_a_wide_weight(P, m, n, k):
    """Up to 32 rows of a weight whose 256-column tiles fill the SMs: tiles of few
    rows, split by columns (N a multiple of 32), and the forms beside them."""
    g = gen(m + n + k)
    q, s = weight(g, n, k)
    x = randn(g, 64, k)
    y = P.ops.fp8_linear(x[:m], q, s)
    check_linear(y, x[:m], q, s)
    assert same_bits(y, P.ops.fp8_linear(x, q, s)[:m])  # the rows of a larger batch: the wide form


def test_linear_leading_dims_pitch_and_no_rows(P):
    g = gen(3)
    q, s = weight(g, 200, 256)
    x = randn(g, 3, 5, 256)
    assert same_bits(P.ops.fp8_linear(x, q, s).view(15, 200), P.ops.fp8_linear(x.view(15, 256), q, s))
    wide = randn(g, 40, 768)
    assert same_bits(P.ops.fp8_linear(wide[:, 256:512], q, s), P.ops.fp8_linear(wide[:, 256:512].contiguous(), q, s))
    assert same_bits(P.ops.fp8_linear(x[0, 0], q, s), P.ops.fp8_linear(x[0, :1], q, s)[0])
    assert P.ops.fp8_linear(x[:0], q, s).shape == (0, 5, 200)


@pytest.mark.parametrize("m", [1, 7, 40, 300])
def test_linear_special_rows(P, m):
    """Rows of zeros give zeros; a NaN or an infinity spoils its row alone."""
    g = gen(m)
    q, s = weight(g, 384, 512)
    x = randn(g, m, 512)
    x[m // 2] = 0
    clean = P.ops.fp8_linear(x, q, s)
    assert torch.equal(clean[m // 2], torch.zeros_like(clean[0]))
    if m > 2:
        x[0, 300] = float("nan")
        x[1, 5] = float("inf")
        x[m - 1, 511] = float("-inf")
        y = P.ops.fp8_linear(x, q, s)
        assert torch.isnan(y[[0, 1, m - 1]]).all()
        keep = [i for i in range(m) if i not in (0, 1, m - 1)]
        assert same_bits(y[keep], clean[keep])


@pytest.mark.parametrize("scale", [1e-30, 1e-14, 1e20])
def test_linear_range(P, scale):
    """Far from one: below 1e-12 a block keeps the scale of 1e-12 and what is
    left of its values."""
    g = gen(11)
    q, s = weight(g, 256, 256)
    x = (torch.randn(20, 256, generator=g) * scale).to(BF16).to(DEV)
    check_linear(P.ops.fp8_linear(x, q, s), x, q, s)


def test_linear_output_of_odd_width_keeps_its_neighbours(P):
    """Nothing is written outside the output rows."""
    g = gen(12)
    q, s = weight(g, 1001, 256)
    x = randn(g, 130, 256)
    lib = P.capi.load()
    size = int(lib.praxis_b200_fp8_linear_workspace_size(130, 1001, 256))
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    buf = torch.full((130 * 1001 + 512,), 7.0, dtype=BF16, device=DEV)
    out = buf[256:-256]
    p = P.ops._p
    P.capi.check(lib.praxis_b200_fp8_linear(p(x), 130, 256, 256, p(q), p(s), 1001, p(out), p(ws), size, 0,
                                            P.ops._stream(x)))
    assert same_bits(out.view(130, 1001), P.ops.fp8_linear(x, q, s))
    assert bool((buf[:256] == 7).all()) and bool((buf[-256:] == 7).all())


def test_linear_refuses_at_the_c_level(P):
    lib, p = P.capi.load(), P.ops._p
    g = gen(13)
    q, s = weight(g, 128, 256)
    x = randn(g, 40, 256)
    out = torch.empty(40, 128, dtype=BF16, device=DEV)
    size = int(lib.praxis_b200_fp8_linear_workspace_size(40, 128, 256))
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)

    def call(rows=40, k=256, ldx=256, n=128, size=size, x=p(x)):
        return lib.praxis_b200_fp8_linear(x, rows, k, ldx, p(q), p(s), n, p(out), p(ws), size, 0, None)

    for kw in (dict(k=250), dict(ldx=252), dict(ldx=128), dict(n=0), dict(rows=-1), dict(size=size - 1), dict(x=None),
               dict(k=0)):
        assert call(**kw) == P.capi.EINVAL, kw
    assert call() == P.capi.OK
    # 2^24 x 2^7 tiles: their numbers would pass 31 bits (refused before anything is read)
    assert call(rows=0x7fffff00, n=32768) == P.capi.EINVAL and b"tiles" in lib.praxis_b200_last_error()
    # up to 8 rows need no workspace
    assert lib.praxis_b200_fp8_linear_workspace_size(8, 128, 256) == 0
    with pytest.raises(ValueError):
        P.ops.fp8_linear(randn(g, 4, 24), *weight(g, 128, 24))


# -- feed-forward ----------------------------------------------------------------

@pytest.mark.parametrize("m,c,f", [(1, 128, 128), (1, 1024, 512), (5, 256, 384), (16, 384, 128), (70, 256, 640),
                                   (128, 512, 256), (300, 640, 384), (1100, 256, 512),
                                   (2600, 128, 1024)])
def test_mlp(P, m, c, f):
    g = gen(m + c + f)
    gu, down = weight(g, 2 * f, c), weight(g, c, f)
    x = randn(g, m, c)
    y = P.ops.fp8_mlp(x, *gu, *down)
    assert rel(y, swiglu64(rows64(x), w64(*gu), w64(*down))) < 1e-2
    out = torch.full_like(x, 3.0)
    assert P.ops.fp8_mlp(x, *gu, *down, out=out) is out and same_bits(out, y)
    assert P.ops.fp8_mlp(x[:0], *gu, *down).shape == (0, c)


@pytest.mark.parametrize("m", [3, 200])
def test_mlp_of_closed_gates(P, m):
    """silu lies between -40 / (1 + e^40) and 0 for gates below -40, and is
    taken as that bound: |h| <= 1.7e-16 |u|, and an output at most the sum of
    |h| |w|, with a rounding each to E4M3 and to bf16 (2^-4 and 2^-8)."""
    c, f = 128, 256
    one = torch.ones(c, dtype=BF16)
    x = (one * 64.0).expand(m, c).contiguous().to(DEV)
    gate_up = torch.cat([torch.full((f, c), -4.0), torch.full((f, c), 4.0)])  # gates -32768, up values 32768
    gu = P.ops.fp8_pack_weights(gate_up.T.contiguous().to(BF16).to(DEV))
    down = P.ops.fp8_pack_weights(torch.ones(f, c, dtype=BF16, device=DEV))
    bound = 40 / (1 + math.exp(40)) * 32768 * f
    y = P.ops.fp8_mlp(x, *gu, *down).double()
    assert float(y.abs().max()) <= bound * (1 + 2**-4) * (1 + 2**-8)
    # NaN stays in its row
    x[1] = float("nan")
    y2 = P.ops.fp8_mlp(x, *gu, *down).double()
    assert bool(y2[1].isnan().all()) and torch.equal(y2[2], y[2])


@pytest.mark.parametrize("m", [3, 20, 200])
def test_mlp_gates_far_below_zero(P, m):
    """Every hidden column of a block has one gate value and u = 2^90, so the block
    is held as 448 times its scale and an output is 128 h of its block. A gate of
    C = 128 columns is off by (C + 4) 2^-23 of itself, which moves h = g e^g u by
    that times |g|; the exponent's rounding and the approximations add
    |g| 2^-24 + 2^-22, the block's scale and sum less than 2^-16, bf16 2^-8."""
    c, values = 128, [-2.0, -39.0, -41.0, -45.0, -64.0, -80.0, -86.0, -120.0]
    f = 128 * len(values)
    x = torch.full((m, c), 64.0, dtype=BF16, device=DEV)
    gate = torch.tensor(values).repeat_interleave(128)[:, None].expand(f, c) / (64 * c)
    gate_up = torch.cat([gate, torch.full((f, c), 2.0**90 / (64 * c))])
    gu = P.ops.fp8_pack_weights(gate_up.T.contiguous().to(BF16).to(DEV))
    pick = torch.zeros(f, c)
    for i in range(len(values)):
        pick[128 * i:128 * (i + 1), 16 * i:16 * (i + 1)] = 1.0
    down = P.ops.fp8_pack_weights(pick.to(BF16).to(DEV))
    g64, u64 = (rows64(x) @ w64(*gu).T).chunk(2, dim=-1)
    h64 = (g64 / (1 + torch.exp(-g64)) * u64)[:, ::128].repeat_interleave(16, 1) * 128
    h64[:, 16 * 7:] = 0  # e^-120 is no 32-bit number
    a = g64[:, ::128].repeat_interleave(16, 1).abs()
    tol = (a * (c + 4) * 2.0**-23 + a * 2.0**-24 + 2.0**-22 + 2.0**-16) * 1.01 + 2.0**-8
    y = P.ops.fp8_mlp(x, *gu, *down).double()
    assert bool(((y - h64).abs() <= tol * h64.abs()).all()), ((y - h64) / h64)[0, ::16]


@pytest.mark.parametrize("m", [3, 20, 200])
def test_mlp_closed_and_overflowing_gates(P, m):
    """Gates of -32768 leave exactly nothing; a gate that overflows to -inf gives
    NaN in its row, as -inf times exp(-inf) does, and nowhere else."""
    c, f = 128, 256
    x = torch.full((m, c), 64.0, dtype=BF16, device=DEV)
    gate_up = torch.cat([torch.full((f, c), -4.0), torch.full((f, c), 2.0**-20)])
    gu = P.ops.fp8_pack_weights(gate_up.T.contiguous().to(BF16).to(DEV))
    down = P.ops.fp8_pack_weights(torch.ones(f, c, dtype=BF16, device=DEV))
    assert not P.ops.fp8_mlp(x, *gu, *down).any()
    x[1] = 2.0**127
    y = P.ops.fp8_mlp(x, *gu, *down)
    assert bool(y[1].isnan().all()) and not y[[0, 2]].any()


def routing(g, t, e, k, kind):
    logits = torch.randn(t, e, generator=g)
    if kind == "skewed":
        logits[: (3 * t) // 4, 1] += 50.0
    elif kind == "few":
        logits[:, k:] -= 100.0  # every token to the same k experts, the others stay empty
    top = logits.topk(k, -1).indices.contiguous()
    gate = torch.softmax(torch.randn(t, k, generator=g), -1).to(BF16)
    return top.to(DEV), gate.to(DEV)


EXPERTS = [(1, 256, 128, 8, 8, ""), (1, 512, 384, 64, 4, ""), (3, 128, 256, 8, 2, "few"), (7, 256, 128, 4, 1, ""),
           (16, 384, 256, 16, 4, "skewed"), (33, 256, 384, 32, 6, ""), (40, 256, 256, 3, 2, "few"),
           (130, 256, 128, 5, 2, "skewed"), (257, 384, 256, 8, 3, ""), (900, 256, 384, 4, 2, ""),
           (1500, 128, 128, 2, 1, "skewed"), (700, 256, 256, 160, 8, ""),
           (4000, 256, 512, 8, 2, "skewed"), (2048, 128, 128, 4, 2, ""), (2049, 128, 128, 4, 2, "few"),
           (9000, 128, 128, 1, 1, ""), (13000, 128, 128, 40, 5, "skewed"), (1, 128, 128, 1024, 8, ""),
           (1500, 128, 128, 1024, 4, ""), (5, 256, 128, 16, 2, ""), (11, 256, 128, 16, 1, "few"),
           (130, 256, 384, 32, 2, "skewed"), (200, 256, 128, 16, 2, "skewed"), (256, 128, 128, 8, 1, ""),
           (257, 128, 128, 8, 1, ""), (136, 128, 128, 1024, 1, ""), (137, 128, 128, 1024, 1, "")]


@pytest.mark.parametrize("t,c,f,e,k,kind", EXPERTS)
def test_experts(P, t, c, f, e, k, kind):
    g = gen(t + c + f + e)
    gu, down = weight(g, e, 2 * f, c), weight(g, e, c, f)
    x = randn(g, t, c)
    top, gate = routing(g, t, e, k, kind)
    y = P.ops.fp8_moe_forward(x, top, gate, *gu, *down, 2.5)
    want = experts64(rows64(x), top, gate, w64(*gu), w64(*down), 2.5)
    assert rel(y, want) < 1e-2
    for i in (0, t - 1):  # no row hides among the others (3x: a row's errors average over fewer values)
        assert rel(y[i:i + 1], want[i:i + 1]) < 3e-2
    assert same_bits(y, P.ops.fp8_moe_forward(x, top, gate, *gu, *down, 2.5))
    shared = randn(g, t, c)
    both = P.ops.fp8_moe_forward(x, top, gate, *gu, *down, 2.5, shared)
    assert torch.equal(both, (y.float() + shared.float()).to(BF16))


@pytest.mark.parametrize("t,c,f", [(40, 256, 128), (100, 640, 384), (128, 1024, 512)])
def test_rows_do_not_depend_on_their_neighbours(P, t, c, f):
    """The same bits in a small batch (few rows per tile) and in a large one."""
    g = gen(t + c)
    gu, down = weight(g, 4, 2 * f, c), weight(g, 4, c, f)
    x = randn(g, 3000, c)
    top, gate = routing(g, 3000, 4, 1, "")
    whole = P.ops.fp8_moe_forward(x, top, gate, *gu, *down, 1.0)
    part = P.ops.fp8_moe_forward(x[:t], top[:t], gate[:t], *gu, *down, 1.0)
    assert same_bits(part, whole[:t])
    dense = [q[0].contiguous() for q in (*gu, *down)]
    assert same_bits(P.ops.fp8_mlp(x[:20], *dense), P.ops.fp8_mlp(x, *dense)[:20])


@pytest.mark.parametrize("t", [1, 900])
def test_more_than_1024_experts_are_refused(P, t):
    c = f = 128
    weights = [torch.zeros(1025, *s, device=DEV).to(d) for s, d in (((2 * f, c), F8), ((2, 1), torch.float32),
                                                                   ((c, f), F8), ((1, 1), torch.float32))]
    top = torch.zeros(t, 2, dtype=torch.int64, device=DEV)
    with pytest.raises(Exception, match="1024 experts"):
        P.ops.fp8_moe_forward(torch.zeros(t, c, dtype=BF16, device=DEV), top, torch.zeros(t, 2, dtype=BF16, device=DEV),
                              *weights, 1.0)


def test_experts_zero_tokens_zero_gates_and_special_rows(P):
    g = gen(21)
    t, c, f, e, k = 50, 256, 128, 8, 2
    gu, down = weight(g, e, 2 * f, c), weight(g, e, c, f)
    x = randn(g, t, c)
    top, gate = routing(g, t, e, k, "")
    assert P.ops.fp8_moe_forward(x[:0], top[:0], gate[:0], *gu, *down, 2.5).shape == (0, c)
    gate[4] = 0
    clean = P.ops.fp8_moe_forward(x, top, gate, *gu, *down, 2.5)
    assert torch.equal(clean[4], torch.zeros_like(clean[4]))
    x[7, 3] = float("nan")
    x[8, 255] = float("inf")
    y = P.ops.fp8_moe_forward(x, top, gate, *gu, *down, 2.5)
    assert torch.isnan(y[7:9]).all()
    keep = [i for i in range(t) if i not in (7, 8)]
    assert same_bits(y[keep], clean[keep])


def test_experts_with_a_repeated_expert(P):
    """A token may name an expert twice: both slots count."""
    g = gen(22)
    t, c, f, e = 9, 256, 128, 4
    gu, down = weight(g, e, 2 * f, c), weight(g, e, c, f)
    x = randn(g, t, c)
    top = torch.full((t, 3), 2, dtype=torch.int64, device=DEV)
    gate = randn(g, t, 3).abs()
    want = experts64(rows64(x), top, gate, w64(*gu), w64(*down), 1.0)
    assert rel(P.ops.fp8_moe_forward(x, top, gate, *gu, *down, 1.0), want) < 1e-2


@pytest.mark.parametrize("t", [5, 300])
def test_experts_out_of_range_index_is_reported(P, t):
    g = gen(23)
    c, f, e, k = 128, 128, 4, 2
    gu, down = weight(g, e, 2 * f, c), weight(g, e, c, f)
    top, gate = routing(g, t, e, k, "")
    top[t // 2, 0] = e + 3
    top[t // 3, 1] = -1
    P.ops.fp8_moe_forward(randn(g, t, c), top, gate, *gu, *down, 1.0)
    assert P.capi.device_error(0) == 4  # kErrIndexRange, clamped


def test_bank_chunks_and_tail(P):
    g = gen(24)
    t, c, f, e, k = 300, 256, 128, 8, 2
    gu = randn(g, e, c, 2 * f, scale=0.02)
    down = randn(g, e, f, c, scale=0.02)
    bank = P.pack_routed_experts_fp8(gu, down)
    codes, scale = quantized(gu.float().mT, 128)
    assert torch.equal(bank.gate_up_q.float(), codes) and torch.equal(bank.gate_up_scale, scale)
    x, shared, residual = randn(g, t, c), randn(g, t, c), randn(g, t, c)
    top, gate = routing(g, t, e, k, "")
    whole = bank.routed_forward(x, top, gate, scaling=2.5, chunk_size=t)
    want = experts64(rows64(x), top, gate, w64(bank.gate_up_q, bank.gate_up_scale), w64(bank.down_q, bank.down_scale),
                     2.5)
    assert rel(whole, want) < 1e-2
    parts = bank.routed_forward(x, top, gate, scaling=2.5, chunk_size=70)
    assert rel(parts, want) < 1e-2
    both = bank.routed_forward_with_shared(x, top, gate, scaling=2.5, chunk_size=t, shared=shared)
    assert torch.equal(both, whole + shared)
    fallback = bank.routed_forward_with_shared(x, top, gate, scaling=2.5, chunk_size=t, shared=shared.float())
    assert torch.equal(fallback, whole + shared.float())
    tail = P.ops.Tail(residual)
    new, normed = bank.routed_forward_tail(x, top, gate, scaling=2.5, chunk_size=t, tail=tail, shared=shared)
    assert normed is None and torch.equal(new, residual + both)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("kind", ["add", "norm", "mod", "mod_unfused", "mod_rows"])
@pytest.mark.parametrize("t,chunk", [(1, 1), (3, 3), (5, 2), (52, 52), (300, 70)])
def test_bank_tail_forms(P, t, chunk, kind, shared):
    """Every form of the fused tail, behind the streaming and the tiled
    products: the bits of the combine of the plain forward's output (one row per
    token, gate 1), which has tests of its own."""
    g = gen(t + 7 * len(kind))
    c, f, e, k = 256, 128, 8, 2
    gu, down = weight(g, e, 2 * f, c), weight(g, e, c, f)
    bank = P.B200FP8RoutedExperts(dict(gate_up_q=gu[0], gate_up_scale=gu[1], down_q=down[0], down_scale=down[1]))
    x, residual = randn(g, t, c), randn(g, t, c)
    sh = randn(g, t, c) if shared else None
    top, gate = routing(g, t, e, k, "")
    tail = P.ops.Tail(residual)
    if kind != "add":
        tail = tail._replace(norm_weight=1 + randn(g, c, scale=0.1, dtype=torch.float32), eps=1e-6, norm_scale=0.8125)
    if kind.startswith("mod"):
        geom = (26, 8, 2, 2, 3, 2) if kind == "mod_rows" else None
        rows = 8 * (-(-t // 26)) if geom else t
        tail = tail._replace(mod=randn(g, rows, 2 * c, scale=0.2), mod_fma=kind != "mod_unfused", mod_geom=geom)
    kw = dict(scaling=2.5, chunk_size=chunk)
    y = (bank.routed_forward(x, top, gate, **kw) if sh is None
         else bank.routed_forward_with_shared(x, top, gate, shared=sh, **kw))
    same = P.ops.dispatch(torch.zeros(t, 1, dtype=torch.int64, device=DEV), torch.ones(t, 1, dtype=BF16, device=DEV), 1)
    rows = torch.zeros(P.ops.padded_rows(t, 1), c, dtype=BF16, device=DEV)
    rows[:t] = y
    want = P.ops.combine_tail(rows, same, 1.0, tail, rows_rescaled=True)
    new, normed = bank.routed_forward_tail(x, top, gate, tail=tail, shared=sh, **kw)
    assert same_bits(new, want[0])
    assert (normed is None and want[1] is None) if kind == "add" else same_bits(normed, want[1])


def test_offsets_past_32_bits(P):
    """Weights of more than 2^32 bytes and activations of more than 2^32."""
    e, c, f = 65, 8192, 4096
    g = torch.Generator(device=DEV).manual_seed(25)

    def bank(*shape):
        q = torch.randint(0, 120, shape, generator=g, device=DEV, dtype=torch.uint8).view(F8)
        return q, torch.rand(shape[0], shape[1] // 128, shape[2] // 128, generator=g, device=DEV) * 1e-4

    gu, down = bank(e, 2 * f, c), bank(e, c, f)
    assert gu[0].numel() > 2**32
    last = tuple(w[e - 1:].contiguous() for w in (*gu, *down))
    for t in (3, 150):
        x = torch.randn(t, c, generator=g, device=DEV).to(BF16)
        top = torch.full((t, 1), e - 1, dtype=torch.int64, device=DEV)
        gate = torch.ones(t, 1, dtype=BF16, device=DEV)
        y = P.ops.fp8_moe_forward(x, top, gate, *gu, *down, 1.0)
        assert same_bits(y, P.ops.fp8_moe_forward(x, top * 0, gate, *last, 1.0)) and bool(y.any())
    del gu, down, last
    rows, k = 2**32 // 8192 + 200, 8192
    x = torch.randn(1000, k, generator=g, device=DEV).to(BF16)
    q, s = weight(gen(26), 24, k)
    big = torch.zeros(rows, k, dtype=BF16, device=DEV)
    big[-1000:] = x
    y = P.ops.fp8_linear(big, q, s)
    check_linear(y[-1000:], x, q, s)
    assert not y[:-1000].any()


# -- the routing -----------------------------------------------------------------

def route64(logits, bias, k, act, groups, top, score):
    """(the picks, the gates, whether a token's choices are apart by 1e-6 at least)."""
    z = logits.double()
    t, e = z.shape
    s = 1 / (1 + torch.exp(-z)) if act == "sigmoid" else torch.softmax(z, -1)
    c = s if bias is None else s + bias.double()
    per = c.view(t, groups, -1).sort(-1, descending=True).values
    of = per[..., :2].sum(-1) if score == "top2" else per[..., 0]
    of, order = of.sort(dim=-1, descending=True, stable=True)
    clear = (of[:, top - 1] - of[:, top] > 1e-6) if top < groups else torch.ones(t, dtype=torch.bool, device=z.device)
    shut = torch.ones(t, groups, dtype=torch.bool, device=z.device).scatter_(1, order[:, :top], False)
    v, idx = c.masked_fill(shut.repeat_interleave(e // groups, 1), -math.inf).sort(dim=-1, descending=True, stable=True)
    gap = v[:, : k + 1].diff(dim=-1).neg() if k < e else v[:, :k].diff(dim=-1).neg()
    if gap.shape[1]:
        clear &= (gap > 1e-6).all(-1)
    idx = idx[:, :k]
    w = s.gather(1, idx)
    return idx, w / w.sum(-1, keepdim=True), clear


ROUTES = [(1, 256, 8, 4, 8), (1, 8, 4, 1, 2), (13, 64, 8, 3, 6), (1000, 256, 8, 4, 8), (513, 96, 6, 3, 6),
          (257, 160, 8, 3, 6), (300, 255, 17, 5, 8), (300, 252, 9, 9, 1), (77, 32, 32, 8, 8), (77, 62, 31, 2, 4),
          (64, 130, 2, 1, 8), (40, 129, 3, 2, 5), (40, 9, 3, 3, 8)]


@pytest.mark.parametrize("act", ["sigmoid", "softmax"])
@pytest.mark.parametrize("score", ["top2", "max"])
@pytest.mark.parametrize("t,e,groups,top,k", ROUTES)
def test_route_groups(P, t, e, groups, top, k, act, score):
    g = gen(t + e + groups)
    logits = torch.randn(t, e, generator=g).to(DEV)
    for bias in (None, (torch.randn(e, generator=g) * 0.1).to(DEV)):
        idx, gate = P.ops.route(logits, bias, k, act, groups=groups, top_groups=top, group_score=score)
        want, w, clear = route64(logits, bias, k, act, groups, top, score)
        # fp32 scores are within 2^-21 of the 64-bit ones: choices further apart than 1e-6 are decided alike
        assert clear.float().mean() > 0.8
        assert torch.equal(idx[clear], want[clear])
        # one bf16 rounding (2^-8), after fp32 quotients (4 roundings of 2^-24 and expf's 2 ulp)
        err = (gate.double() - w)[clear].abs()
        assert (err <= (2.0**-8 + 2.0**-20) * w[clear]).all()
        assert idx.dtype == torch.int64 and gate.dtype == BF16
        assert (idx.sort(-1).values.diff(dim=-1) > 0).all() and idx.min() >= 0 and idx.max() < e


def test_route_groups_ties_go_to_the_lower_index(P):
    g = gen(31)
    logits = torch.randint(0, 3, (400, 64), generator=g).float().to(DEV)
    idx, _ = P.ops.route(logits, None, 6, "sigmoid", groups=8, top_groups=3, group_score="max")
    want, _, _ = route64(logits, None, 6, "sigmoid", 8, 3, "max")
    assert torch.equal(idx, want)
    idx, gate = P.ops.route(torch.zeros(3, 64, device=DEV), None, 4, "softmax", groups=8, top_groups=2)
    assert torch.equal(idx, torch.arange(4, device=DEV).expand(3, 4)) and bool((gate == 0.25).all())


@pytest.mark.parametrize("score", ["top2", "max"])
@pytest.mark.parametrize("t,e,groups,top,k", ROUTES)
def test_route_groups_many_ties(P, t, e, groups, top, k, score):
    g = gen(t + e)
    logits = torch.randint(0, 2, (t, e), generator=g).float().to(DEV)
    idx, gate = P.ops.route(logits, None, k, "sigmoid", groups=groups, top_groups=top, group_score=score)
    want, want_gate, _ = route64(logits, None, k, "sigmoid", groups, top, score)
    assert torch.equal(idx, want)
    assert bool(((gate.double() - want_gate).abs() <= 1.01 * 2**-8 * want_gate).all())


@pytest.mark.parametrize("e,groups", [(256, 8), (64, 4), (130, 2)])
def test_route_groups_unaligned_rows_and_bias(P, e, groups):
    g = gen(e)
    logits, bias = torch.randn(50, e, generator=g).to(DEV), torch.randn(e, generator=g).to(DEV)
    run = lambda lo, bi: P.ops.route(lo, bi, 6, groups=groups, top_groups=2)  # noqa: E731
    shift = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)  # noqa: E731
    want = run(logits, bias)
    for other in (run(shift(logits), bias), run(logits, shift(bias)), run(shift(logits), shift(bias))):
        assert torch.equal(other[0], want[0]) and same_bits(other[1], want[1])


@pytest.mark.parametrize("act", ["sigmoid", "softmax"])
def test_route_groups_masked_experts(P, act):
    """Masked experts (-inf) are picked last; a row with nothing left has
    gates of zero and the lowest experts; NaN stays inside the range."""
    g = gen(32)
    logits = torch.randn(6, 32, generator=g)
    logits[0] = -math.inf
    logits[1, 3:] = -math.inf
    logits[2] = torch.finfo(torch.float32).min
    logits[3, ::2] = -math.inf
    logits[4, 5] = float("nan")
    logits[5] = float("nan")
    idx, gate = P.ops.route(logits.to(DEV), None, 4, act, groups=4, top_groups=2)
    assert torch.equal(idx[0].cpu(), torch.arange(4)) and bool((gate[0] == 0).all())
    assert set(idx[1].tolist()) == {0, 1, 2, 3} and float(gate[1][idx[1] == 3]) == 0.0
    assert abs(float(gate[1].float().sum()) - 1) < 4 * 2.0**-8
    if act == "sigmoid":
        assert bool((gate[2] == 0).all())
    else:
        assert bool((gate[2] == 0.25).all())
    assert bool((idx[3] % 2 == 1).all())
    assert bool(((idx >= 0) & (idx < 32)).all()) and bool((idx.sort(-1).values.diff(dim=-1) > 0).all())


def test_route_groups_bias_only_chooses(P):
    logits = torch.zeros(1, 16, device=DEV)
    bias = torch.zeros(16, device=DEV)
    bias[13], bias[2] = 5.0, -math.inf
    idx, gate = P.ops.route(logits, bias, 2, "sigmoid", groups=4, top_groups=1, group_score="max")
    assert idx.tolist() == [[13, 12]] and gate.tolist() == [[0.5, 0.5]]
    idx, _ = P.ops.route(logits, bias, 4, "sigmoid", groups=4, top_groups=4)
    assert 2 not in idx[0].tolist()


def test_route_groups_no_tokens_and_refusals(P):
    idx, gate = P.ops.route(torch.zeros(0, 32, device=DEV), None, 4, groups=4, top_groups=2)
    assert idx.shape == (0, 4) and gate.shape == (0, 4)
    lib, p = P.capi.load(), P.ops._p
    x = torch.zeros(2, 256, device=DEV)
    top, gate = torch.empty(2, 16, dtype=torch.int64, device=DEV), torch.empty(2, 16, dtype=BF16, device=DEV)
    for e, k, act, groups, open_, score in ((257, 8, 0, 1, 1, 0), (256, 9, 0, 8, 4, 0), (256, 8, 2, 8, 4, 0),
                                            (256, 8, 0, 7, 4, 0), (256, 8, 0, 64, 4, 0), (256, 8, 0, 8, 9, 0),
                                            (256, 8, 0, 8, 4, 2), (256, 8, 0, 32, 0, 0), (32, 8, 0, 8, 1, 0)):
        assert lib.praxis_b200_route_groups(p(x), None, 2, e, k, act, groups, open_, score, p(top), p(gate), 0,
                                            None) == P.capi.EINVAL


# -- streams, graphs, together -----------------------------------------------------

def layer(P, g, dim=256, hidden=128, e=32, k=4):
    m = P.B200MoEFeedForward(dim, hidden, e, k, 2.5, router_groups=4, router_top_groups=2).to(DEV)
    with torch.no_grad():
        m.router.weight.copy_(randn(g, e, dim, scale=0.2, dtype=torch.float32))
        m.expert_bias.copy_(torch.randn(e, generator=g) * 0.1)
        m.shared.gate_up.copy_(randn(g, dim, 2 * hidden, scale=0.02))
        m.shared.down.copy_(randn(g, hidden, dim, scale=0.02))
    m.shared.to(BF16)
    m.set_routed_weights(randn(g, e, dim, 2 * hidden, scale=0.02), randn(g, e, hidden, dim, scale=0.02), "fp8")
    m.quantize_shared()
    return m


@pytest.mark.parametrize("t", [1, 19, 400])
def test_layer_with_groups_and_fp8_experts(P, t):
    """Router, groups, routed and shared experts together, as a model uses them."""
    g = gen(40 + t)
    m = layer(P, g)
    x = randn(g, 1, t, 256)
    y = m(x)
    assert y.shape == x.shape
    flat = x.view(t, 256)
    logits = P.ops.router_logits(flat, m.router_terms())[0]
    assert rel(logits, flat.double() @ m.router.weight.detach().double().T) < 1e-5
    top, gate = m.route(flat)
    want_top, _, clear = route64(logits, m.expert_bias, 4, "sigmoid", 4, 2, "top2")
    assert torch.equal(top[clear], want_top[clear])
    b, s = m.routed, m.shared
    want = experts64(rows64(flat), top, gate, w64(b.gate_up_q, b.gate_up_scale), w64(b.down_q, b.down_scale), 2.5)
    want = want + swiglu64(rows64(flat), w64(s.gate_up_q, s.gate_up_scale), w64(s.down_q, s.down_scale))
    # the shared expert's row and the sum with it are rounded too: two more of 2^-8 / sqrt(3)
    assert rel(y.view(t, 256), want) < 1.1e-2
    residual = randn(g, 1, t, 256)
    new, _ = m.forward_tail(x, residual)
    assert torch.equal(new, residual + y)
    pair = m.forward_pair([x, x])
    assert same_bits(pair[0], y) and same_bits(pair[1], y)


def test_other_stream(P):
    g = gen(50)
    m = layer(P, g)
    x = randn(g, 200, 256)
    want = m(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = m(x)
        lin = P.ops.fp8_linear(x, m.shared.gate_up_q, m.shared.gate_up_scale)
    side.synchronize()
    assert same_bits(got, want) and same_bits(lin, P.ops.fp8_linear(x, m.shared.gate_up_q, m.shared.gate_up_scale))


def test_two_streams_at_once(P):
    g = gen(51)
    q, s = weight(g, 1024, 512)
    xs = [randn(g, m, 512) for m in (3, 700)]
    want = [P.ops.fp8_linear(x, q, s) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(20):
        for i, (x, stream) in enumerate(zip(xs, streams, strict=True)):
            with torch.cuda.stream(stream):
                got[i].append(P.ops.fp8_linear(x, q, s))
    torch.cuda.synchronize()
    assert all(same_bits(y, w) for ys, w in zip(got, want, strict=True) for y in ys)


@pytest.mark.parametrize("t", [1, 12, 300])
def test_two_captured_graphs_and_eager_calls(P, t):
    g = gen(60 + t)
    m = layer(P, g)
    q, s = m.shared.gate_up_q, m.shared.gate_up_scale
    xs = [randn(g, t, 256) for _ in range(4)]
    want = [(m(x).clone(), P.ops.fp8_linear(x, q, s).clone()) for x in xs]
    graphs, ins, outs = [], [], []
    for _ in range(2):
        buf = torch.zeros_like(xs[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((m(buf), P.ops.fp8_linear(buf, q, s)))
        graphs.append(graph)
        ins.append(buf)
    for i, j in ((0, 1), (2, 3), (1, 0)):
        ins[0].copy_(xs[i])
        ins[1].copy_(xs[j])
        graphs[0].replay()
        graphs[1].replay()
        eager = m(xs[i])
        for got, w in zip((*outs[0], *outs[1], eager), (*want[i], *want[j], want[i][0]), strict=True):
            assert same_bits(got, w)


@pytest.mark.parametrize("t", [1, 5, 48, 700, 2500])
def test_calls_in_a_row_see_each_others_results(P, t):
    """Inputs, routing and weights written by the call right before: the same
    bits queued back to back, captured, and with a wait after every call."""
    g = gen(90 + t)
    c, f, e, k = 256, 384, 8, 2
    banks = [(randn(g, e, c, 2 * f, scale=0.06), randn(g, e, f, c, scale=0.06)) for _ in range(3)]
    square = randn(g, c, c, scale=0.06)
    x0 = randn(g, t, c)
    router = randn(g, e, c, dtype=torch.float32)
    terms = P.ops.split_router_weight(router)

    def chain(after=lambda: None):
        x = x0
        for gate_up, down in banks:
            w = P.ops.fp8_pack_weights(square)
            after()
            x = P.ops.fp8_linear(x, *w)
            after()
            top, gate = P.ops.route(P.ops.router_logits(x, terms)[0], None, k, groups=4, top_groups=2)
            after()
            gu, dn = P.ops.fp8_pack_weights(gate_up), P.ops.fp8_pack_weights(down)
            after()
            x = x + P.ops.fp8_moe_forward(x, top, gate, *gu, *dn, 1.0)
            after()
            x = P.ops.fp8_mlp(x, *(q[0] for q in gu), *(q[0] for q in dn))
            after()
        return x

    want = chain(torch.cuda.synchronize)
    for _ in range(5):
        assert same_bits(chain(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for _ in range(5):
        got.zero_()
        graph.replay()
        assert same_bits(got, want)


@pytest.mark.parametrize("t", [1, 70])
@torch.no_grad()
def test_captured_layer(P, t):
    """The graph pool finds layers with FP8 experts and replays their forward."""
    g = gen(80 + t)
    m = layer(P, g).eval().requires_grad_(False)
    xs = [randn(g, 1, t, 256) for _ in range(3)]
    want = [m(x) for x in xs]
    pool = P.graphs.enable_moe_cuda_graphs(torch.nn.ModuleList([m]), warmup=1)
    try:
        for x, y in zip(xs, want, strict=True):
            assert same_bits(m(x), y)
        assert [s["captures"] for s in pool.stats().values()] == [1]
    finally:
        pool.release()


def test_torch_operators_match_direct_calls(P):
    g = gen(70)
    t, c, f, e, k = 30, 256, 128, 8, 2
    gu, down, lin = weight(g, e, 2 * f, c), weight(g, e, c, f), weight(g, 300, c)
    x, logits = randn(g, t, c), randn(g, t, e, dtype=torch.float32)
    ns, ops = torch.ops.praxis_b200, P.ops
    top, gate = ns.route_groups(logits, None, k, "softmax", 4, 2, "max")
    want = ops.route(logits, None, k, "softmax", groups=4, top_groups=2, group_score="max")
    assert torch.equal(top, want[0]) and same_bits(gate, want[1])
    assert same_bits(ns.fp8_linear(x, *lin), ops.fp8_linear(x, *lin))
    dense = (gu[0][0], gu[1][0], down[0][0], down[1][0])
    assert same_bits(ns.fp8_mlp(x, *dense), ops.fp8_mlp(x, *dense))
    assert same_bits(ns.fp8_moe_forward(x, top, gate, *gu, *down, 2.5, None),
                     ops.fp8_moe_forward(x, top, gate, *gu, *down, 2.5))
    torch.library.opcheck(ns.route_groups.default, (logits, None, k, "softmax", 4, 2, "max"),
                          test_utils=("test_schema", "test_faketensor"))
    # (the schema check multiplies its arguments, which torch cannot do in E4M3)
    for op, args in ((ns.fp8_linear, (x, *lin)), (ns.fp8_mlp, (x, *dense)),
                     (ns.fp8_moe_forward, (x, top, gate, *gu, *down, 2.5, None))):
        torch.library.opcheck(op.default, args, test_utils=("test_faketensor",))


@pytest.mark.parametrize("t,e,k", [(9, 160, 4), (40, 1024, 2), (1, 1024, 8), (150, 1024, 1), (17, 96, 8)])
def test_few_slots_of_many_experts_stay_inside_their_workspace(P, t, e, k):
    """Slots all on different experts (as far as they go): the most tiles that a
    call can have. Nothing behind the workspace's stated size is written."""
    g = gen(t + e)
    c, f = 256, 128
    gu, down = weight(g, e, 2 * f, c), weight(g, e, c, f)
    x = randn(g, t, c)
    top = (torch.arange(t * k).view(t, k) * 7 % e).to(DEV)
    gate = randn(g, t, k).abs()
    lib = P.capi.load()
    size = lib.praxis_b200_fp8_ffn_workspace_size(t, k, e, c, f)
    ws = torch.full((size + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
    out = torch.empty_like(x)
    args = P.capi.Fp8FfnArgs(
        x=x.data_ptr(), top_idx=top.data_ptr(), gate=gate.data_ptr(), out=out.data_ptr(), gate_up_q=gu[0].data_ptr(),
        gate_up_scale=gu[1].data_ptr(), down_q=down[0].data_ptr(), down_scale=down[1].data_ptr(), tokens=t, dim=c,
        hidden=f, experts=e, top_k=k, scaling=1.0, workspace=ws.data_ptr(), workspace_size=size, device=0,
        stream=torch.cuda.current_stream().cuda_stream)
    P.capi.check(lib.praxis_b200_fp8_ffn(args))
    assert bool((ws[size:] == 0xA5).all())
    want = experts64(rows64(x), top, gate, w64(*gu), w64(*down), 1.0)
    assert rel(out, want) < 1e-2
    assert same_bits(out, P.ops.fp8_moe_forward(x, top, gate, *gu, *down, 1.0))
