"""Every product kernel of the linear layers - tile, direction, gate, sums, split, operand over its end - against the definition in
64 bits, exactly.

Operands are small whole numbers and the slope is 1/4, so every product and every sum of them (below 2^22, in quarters) is exact
in float32 whatever the order: a kernel's result is the definition's, rounded once to the output's type, and one element in the
wrong place or left out shows.  The sizes are among the smallest at which the choice of kernels takes the named one;
sg2im_linear_plan says which one that is, and a change of the choice that drops one of them fails the first test."""
import ctypes

import pytest
import torch

gpu = pytest.mark.gpu
F64, F32, BF16 = torch.float64, torch.float32, torch.bfloat16
SLOPE = 0.25
FORWARD, DX, DW = 0, 1, 2

# bfloat16?, direction, gated, with sums, tile, reduction split, (rows, k, n)
CASES = [
  (0, FORWARD, 0, 0, 16, 0, (256, 256, 256)), (0, FORWARD, 0, 0, 64, 0, (256, 256, 1280)), (0, FORWARD, 0, 0, 64, 0, (90, 3, 130)),
  (0, FORWARD, 0, 0, 64, 1, (512, 768, 512)), (0, FORWARD, 0, 0, 64, 1, (354, 631, 722)), (0, FORWARD, 0, 0, 128, 0, (1792, 256, 1792)),
  (0, FORWARD, 0, 0, 128, 0, (25141, 4, 68)), (0, FORWARD, 0, 0, 128, 1, (768, 1536, 1536)), (0, FORWARD, 0, 0, 128, 1, (2122, 3718, 85)),
  (0, FORWARD, 0, 0, 128, 0, (3200, 512, 1152)), (0, FORWARD, 0, 0, 256, 1, (14080, 5376, 768)),
  (0, DX, 0, 0, 64, 0, (256, 256, 256)), (0, DX, 0, 0, 64, 1, (256, 256, 512)), (0, DX, 0, 0, 64, 1, (70, 33, 261)),
  (0, DX, 0, 0, 128, 0, (1792, 1792, 256)), (0, DX, 0, 0, 128, 0, (25401, 65, 2)), (0, DX, 0, 0, 128, 1, (768, 1536, 1536)),
  (0, DX, 0, 0, 128, 1, (9656, 81, 852)), (0, DX, 0, 0, 256, 1, (6144, 1792, 5376)),
  (0, DX, 1, 0, 64, 0, (256, 256, 256)), (0, DX, 1, 0, 64, 1, (256, 256, 512)), (0, DX, 1, 0, 64, 1, (70, 33, 261)),
  (0, DX, 1, 0, 128, 0, (1792, 1792, 256)), (0, DX, 1, 0, 128, 0, (25401, 65, 2)), (0, DX, 1, 0, 128, 1, (768, 1536, 1024)),
  (0, DX, 1, 0, 128, 1, (8364, 67, 560)),
  (0, DW, 0, 0, 64, 0, (256, 256, 256)), (0, DW, 0, 0, 64, 1, (512, 256, 256)), (0, DW, 0, 0, 64, 1, (4099, 161, 515)),
  (0, DW, 0, 0, 128, 0, (256, 1792, 1792)), (0, DW, 0, 0, 128, 0, (4, 390, 7210)), (0, DW, 0, 0, 128, 1, (1536, 768, 1536)),
  (0, DW, 0, 0, 128, 1, (934, 198, 4221)), (0, DW, 0, 0, 256, 1, (5376, 5888, 1792)),
  (0, DW, 0, 1, 64, 0, (256, 256, 256)), (0, DW, 0, 1, 64, 1, (4099, 161, 515)), (0, DW, 0, 1, 128, 0, (256, 1792, 1792)),
  (0, DW, 0, 1, 128, 1, (1024, 256, 4352)), (0, DW, 0, 1, 128, 1, (922, 2760, 323)),
  (0, DW, 1, 1, 64, 0, (256, 256, 256)), (0, DW, 1, 1, 64, 1, (4099, 161, 515)), (0, DW, 1, 1, 128, 0, (4, 390, 7210)),
  (0, DW, 1, 1, 128, 1, (1024, 1536, 768)), (0, DW, 1, 1, 128, 1, (4097, 1372, 73)),
  (1, FORWARD, 0, 0, 16, 0, (256, 256, 256)), (1, FORWARD, 0, 0, 64, 0, (768, 256, 256)), (1, FORWARD, 0, 0, 64, 0, (90, 7, 130)),
  (1, FORWARD, 0, 0, 64, 1, (256, 3840, 256)), (1, FORWARD, 0, 0, 64, 1, (584, 1451, 269)), (1, FORWARD, 0, 0, 128, 0, (1792, 256, 1792)),
  (1, FORWARD, 0, 0, 128, 0, (32701, 1000, 260)), (1, FORWARD, 0, 0, 128, 1, (4352, 3328, 256)), (1, FORWARD, 0, 0, 128, 1, (65, 7515, 2081)),
  (1, FORWARD, 0, 0, 256, 0, (2560, 256, 3328)), (1, FORWARD, 0, 0, 256, 0, (2741, 64, 2949)), (1, FORWARD, 0, 0, 256, 1, (3328, 4096, 1280)),
  (1, FORWARD, 0, 0, 256, 1, (1517, 4416, 2924)), (1, FORWARD, 0, 0, 256, 0, (131072, 64, 256)),
  (1, DX, 0, 0, 64, 0, (256, 256, 256)), (1, DX, 0, 0, 64, 1, (256, 256, 1280)), (1, DX, 0, 0, 64, 1, (70, 33, 822)),
  (1, DX, 0, 0, 128, 0, (1792, 1792, 256)), (1, DX, 0, 0, 128, 0, (32701, 1000, 260)), (1, DX, 0, 0, 128, 1, (4352, 256, 3328)),
  (1, DX, 0, 0, 128, 1, (66, 6347, 3302)), (1, DX, 0, 0, 256, 0, (3328, 2560, 256)), (1, DX, 0, 0, 256, 0, (32701, 1024, 256)),
  (1, DX, 0, 0, 256, 1, (1280, 3328, 4096)),
  (1, DX, 1, 0, 64, 0, (256, 256, 256)), (1, DX, 1, 0, 64, 1, (256, 256, 768)), (1, DX, 1, 0, 64, 1, (8, 33, 457)),
  (1, DX, 1, 0, 128, 0, (1792, 1792, 256)), (1, DX, 1, 0, 128, 0, (32701, 1000, 260)), (1, DX, 1, 0, 128, 1, (768, 256, 7424)),
  (1, DX, 1, 0, 128, 1, (2122, 65, 3200)),
  (1, DW, 0, 0, 64, 0, (256, 256, 256)), (1, DW, 0, 0, 64, 1, (1280, 256, 256)), (1, DW, 0, 0, 64, 1, (4099, 161, 515)),
  (1, DW, 0, 0, 128, 0, (256, 1792, 1792)), (1, DW, 0, 0, 128, 0, (4, 390, 7210)), (1, DW, 0, 0, 128, 1, (3328, 256, 4352)),
  (1, DW, 0, 0, 128, 1, (37510, 322, 68)), (1, DW, 0, 0, 256, 0, (256, 2560, 3328)), (1, DW, 0, 0, 256, 1, (4352, 1536, 2816)),
  (1, DW, 0, 1, 64, 0, (256, 256, 256)), (1, DW, 0, 1, 64, 1, (4099, 161, 515)), (1, DW, 0, 1, 128, 0, (256, 1792, 1792)),
  (1, DW, 0, 1, 128, 1, (6144, 768, 512)), (1, DW, 0, 1, 128, 1, (8492, 1366, 70)), (1, DW, 0, 1, 128, 1, (32768, 1024, 256)),
  (1, DW, 1, 1, 64, 0, (256, 256, 256)), (1, DW, 1, 1, 64, 1, (4099, 161, 515)), (1, DW, 1, 1, 64, 1, (131072, 64, 256)),
  (1, DW, 1, 1, 128, 0, (4, 390, 7210)), (1, DW, 1, 1, 128, 1, (7424, 768, 256)), (1, DW, 1, 1, 128, 1, (36617, 69, 138)),
]


def plan(bf16, which, gated, sums, size):
  from sg2im_amd import _lib
  tile, splits = ctypes.c_int(), ctypes.c_int()
  assert _lib.load().sg2im_linear_plan(*size, bf16, which, gated, sums, ctypes.byref(tile), ctypes.byref(splits)) == _lib.SG2IM_OK
  return tile.value, splits.value


def edges(which, tile, size):
  """is there an operand that ends inside a tile or a chunk of the reduction?"""
  rows, k, n = size
  i, j, r = ((rows, n, k), (rows, k, n), (n, k, rows))[which]
  return bool(i % tile or j % tile or r % 64)


def test_the_sizes_of_this_file_take_every_kernel():
  got, whole = set(), set()
  for bf16, which, gated, sums, tile, split, size in CASES:
    t, s = plan(bf16, which, gated, sums, size)
    assert (t, int(s > 1)) == (tile, split), (bf16, which, gated, sums, size, t, s)
    got.add((bf16, which, gated, sums, tile, split))
    whole.add((bf16, which, gated, sums, tile, edges(which, tile, size)))
  forms = [(FORWARD, 0, 0), (DX, 0, 0), (DX, 1, 0), (DW, 0, 0), (DW, 0, 1), (DW, 1, 1)]
  for bf16 in (0, 1):
    assert (bf16, FORWARD, 0, 0, 16, 0) in got
    for f in forms:
      for tile in (64, 128):
        assert (bf16,) + f + (tile, 0) in got and (bf16,) + f + (tile, 1) in got, (bf16, f, tile)
        assert (bf16,) + f + (tile, True) in whole, (bf16, f, tile)
        assert tile == 64 or f[1] or f[2] or (bf16,) + f + (tile, False) in whole, (bf16, f, tile)
      if not f[1] and not f[2]:
        assert (bf16,) + f + (256, 1) in got and (not bf16 or (bf16,) + f + (256, 0) in got), (bf16, f)


def test_the_plan_is_refused_like_the_calls():
  from sg2im_amd import _lib
  lib = _lib.load()
  t, s = ctypes.c_int(), ctypes.c_int()
  ok = (4, 8, 8, 0, 0, 0, 0, ctypes.byref(t), ctypes.byref(s))
  assert lib.sg2im_linear_plan(*ok) == _lib.SG2IM_OK
  for at, bad in ((0, 0), (0, -1), (0, 1 << 31), (1, 0), (2, 0), (2, (1 << 22) + 1), (3, 2), (4, 3), (4, -1), (7, None), (8, None)):
    assert lib.sg2im_linear_plan(*(ok[:at] + (bad,) + ok[at + 1:])) == _lib.SG2IM_ERR_ARG, (at, bad)


def whole_numbers(seed):
  g = torch.Generator(device='cuda').manual_seed(seed)
  return lambda *s: torch.randint(-2, 3, s, device='cuda', generator=g).to(F32)


def words(bits):
  """truth values (rows, n) as the forward pass keeps them: bit j of word w is column 32 w + j"""
  rows, n = bits.shape
  pad = torch.zeros(rows, -n % 32, dtype=torch.bool, device=bits.device)
  w = torch.cat([bits, pad], 1).view(rows, -1, 32).long()
  w = (w << torch.arange(32, device=bits.device)).sum(2)
  return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def product(a, b):
  """a b in 64 bits, rows at a time (a row of tiles has the same columns, so memory goes by them)"""
  a, b = a.to(F64), b.to(F64).contiguous()
  return torch.cat([part @ b for part in a.split(16384)])


def exactly(got, want, what):
  if not torch.equal(got, want.to(got.dtype)):
    bad = got.to(F64) != want.to(got.dtype).to(F64)
    k = bad.nonzero()[0].tolist()
    raise AssertionError('%s: %d of %d differ, first at %s: %r, want %r' % (what, int(bad.sum()), bad.numel(), k, float(got[tuple(k)]), float(want[tuple(k)])))


@gpu
@pytest.mark.parametrize('bf16,which,gated,sums,tile,split,size', CASES,
                         ids=['%s-%s%s%s-tile%d%s-%s' % ('bf16' if c[0] else 'f32', ('forward', 'dx', 'dw')[c[1]], '-gated' if c[2] else '',
                                                        '-sums' if c[3] else '', c[4], '-split' if c[5] else '', 'x'.join(map(str, c[6]))) for c in CASES])
def test_product(bf16, which, gated, sums, tile, split, size):
  from sg2im_amd import ops
  rows, k, n = size
  t = BF16 if bf16 else F32
  r = whole_numbers(rows + k + n)
  if which == FORWARD:
    x, w, b = r(rows, k).to(t), r(n, k).to(t), r(n).to(t)
    z = product(x, w.t()) + b.to(F64)
    y = torch.where(z > 0, z, z * SLOPE)
    for out in ((F32, BF16) if bf16 else (F32,)):
      res = r(rows, n).to(out)
      got, signs = ops.linear_forward(x, w, b, res, SLOPE, out, signs=True)
      exactly(got, y + res.to(F64), 'y')
      exactly(signs, words(z > 0), 'signs')
    exactly(ops.linear_forward(x, w, None, None, 1.0)[0], z - b.to(F64), 'z')
    return
  dy = r(rows, n).to(t)
  bits = torch.rand(rows, n, device='cuda') < 0.5 if gated else None
  dz = dy.to(F64) * torch.where(bits, 1.0, SLOPE) if gated else dy.to(F64)
  signs = words(bits) if gated else None
  if which == DX:
    w = r(n, k).to(t)
    exactly(ops.linear_backward_data(dy, w, signs, SLOPE), product(dz, w), 'dx')
    return
  x = r(rows, k).to(t)
  want, want_sums = product(dz.t(), x), dz.sum(0)
  start, start_sums = r(n, k), r(n)
  for kept in (x, ops.pack8(x)):                       # (whole numbers up to 2 are exact in 8 bits)
    for out in ((F32, BF16) if bf16 else (F32,)):
      for add in (False, True):
        dw, db = start.to(out, copy=True), start_sums.clone()
        ops.linear_backward_weight(dy, kept, dw, add, db if sums else None, add, signs, SLOPE)
        exactly(dw, want + start.to(F64) if add else want, 'dweight')
        if sums:
          exactly(db, want_sums + start_sums.to(F64) if add else want_sums, 'dbias')


# bfloat16?, gated, bias, dx wanted, dW wanted, (rows, k, n): the gate and the bias gradient go first, in a pass of their own
FIRST = [(0, 1, 1, 1, 1, (676, 1558, 758)), (0, 1, 0, 1, 0, (772, 2521, 1039)), (0, 0, 1, 1, 1, (127110, 1028, 1)), (0, 1, 1, 0, 1, (172314, 146, 1)),
         (1, 1, 1, 1, 1, (5000, 700, 900)), (1, 1, 0, 1, 0, (472, 2108, 1553)), (1, 0, 1, 1, 1, (141264, 778, 1)), (1, 1, 1, 0, 1, (195506, 131, 2)),
         (1, 1, 1, 1, 1, (32768, 1024, 256))]
# ... and where the products do both as they read dy
ITSELF = [(0, 1, 1, 1, 1, (3200, 512, 1152)), (1, 1, 1, 1, 1, (4099, 161, 515)), (1, 0, 1, 1, 1, (32768, 1024, 256)), (1, 1, 1, 1, 1, (131072, 64, 256))]


def test_both_orders_of_the_backward_pass_are_chosen():
  from sg2im_amd import _lib
  first = _lib.load().sg2im_linear_backward_act_first
  for want, cases in ((1, FIRST), (0, ITSELF)):
    for bf16, gated, bias, dx, dw, size in cases:
      assert first(*size, bf16, gated, bias, dx, dw) == want, (bf16, gated, bias, dx, dw, size)


@gpu
@pytest.mark.parametrize('checkpoint8', [False, True])
@pytest.mark.parametrize('bf16,gated,bias,dx,dw,size', FIRST + ITSELF)
def test_training_pass(bf16, gated, bias, dx, dw, size, checkpoint8):
  from sg2im_amd import functional as HF
  rows, k, n = size
  t = BF16 if bf16 else F32
  r = whole_numbers(rows + k + n)
  slope = SLOPE if gated else 1.0
  x, w, b = r(rows, k).to(t).requires_grad_(bool(dx)), r(n, k).to(t).requires_grad_(bool(dw)), r(n).to(t).requires_grad_(bool(bias))
  res = r(rows, n).to(t)
  y = HF.LinearResidual.apply(x, w, b, res, slope, checkpoint8)
  z = product(x.detach(), w.detach().t()) + b.detach().to(F64)
  exactly(y.detach(), torch.where(z > 0, z, z * slope) + res.to(F64), 'y')
  dy = r(rows, n).to(t)
  dz = dy.to(F64) * torch.where(z > 0, 1.0, slope)
  leaves = [p for p in (x, w, b) if p.requires_grad]
  grads = dict(zip([name for name, p in (('dx', x), ('dweight', w), ('dbias', b)) if p.requires_grad], torch.autograd.grad(y, leaves, dy)))
  if dx:
    exactly(grads['dx'], product(dz, w.detach()), 'dx')
  if dw:
    exactly(grads['dweight'], product(dz.t(), x.detach()), 'dweight')
  if bias:
    exactly(grads['dbias'], dz.sum(0), 'dbias')


# the widest operands (2^22 columns), with ones and minus ones: sums stay below 2^24
@gpu
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('size', [(3, 1 << 22, 2), (2, 3, 1 << 22), (1, (1 << 22) - 3, 1), (5, 1, (1 << 22) - 1)])
def test_the_widest_layers(size, dtype):
  from sg2im_amd import functional as HF
  rows, k, n = size
  g = torch.Generator(device='cuda').manual_seed(k + n)
  r = lambda *s: (torch.randint(0, 2, s, device='cuda', generator=g) * 2 - 1).to(dtype)  # noqa: E731
  for slope, checkpoint8 in ((SLOPE, False), (1.0, True)):
    x, w, b, res = [t.requires_grad_(True) for t in (r(rows, k), r(n, k), r(n), r(rows, n))]
    y = HF.LinearResidual.apply(x, w, b, res, slope, checkpoint8)
    z = x.detach().to(F64) @ w.detach().to(F64).t() + b.detach().to(F64)
    exactly(y.detach(), torch.where(z > 0, z, z * slope) + res.detach().to(F64), 'y')
    dy = r(rows, n)
    dz = dy.to(F64) * torch.where(z > 0, 1.0, slope)
    dx, dw, db, dres = torch.autograd.grad(y, (x, w, b, res), dy)
    exactly(dx, dz @ w.detach().to(F64), 'dx')
    exactly(dw, dz.t() @ x.detach().to(F64), 'dweight')
    exactly(db, dz.sum(0), 'dbias')
    exactly(dres, dy, 'dresidual')
