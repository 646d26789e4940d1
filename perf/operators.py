"""What is measured of two operators that a training step of the policy/value networks is made of: the group norm that
carries an activation and a residual sum (channels last), and the AdamW step over all of a network's tensors with its
moments in 32 or in 8 bits.  `run` computes them in their plain form, or with the framework's kernels where `own` is set.

Formulas, x of [N, C, H, W] with C in G groups, n = H * W * C / G values per sample and group:
    mean = sum(x) / n        var = sum((x - mean)^2) / n        rstd = 1 / sqrt(var + eps)
    z = (x - mean) * rstd * weight[c] + bias[c] (+ residual)    y = act(z), act: none, relu, silu(z) = z / (1 + exp(-z))
    dz = dy * act'(z) (relu: 1 where z > 0)                     dresidual = dz
    dbias[c] = sum(dz)       dweight[c] = sum(dz * xhat)        with xhat = (x - mean) * rstd, sums over N, H, W
    dx = rstd * (a - mean_group(a) - xhat * mean_group(a * xhat))  with a = dz * weight[c]

AdamW, step t = t + 1, every product and sum of the moments rounded to 32 bits in this order:
    m = (b1 * m) + ((1 - b1) * g)       v = (b2 * v) + ((1 - b2) * (g * g))
    p = p * (1 - lr * wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
with bfloat16 parameters p is a master copy in 32 bits and the parameter its rounding.  All tensors lie behind each
other in one buffer, each from a multiple of 256 elements on, the gaps zero.  A moment in 8 bits is, for a block of
256 elements, the 11 leading bits `top` (exponent and 3 bits of mantissa) of its largest magnitude, rounded up, and
for each element how many steps of such leading bits below `top` its own are: m a sign and 7 bits (0: zero, k:
leading bits top - 127 + k), v 8 bits (top - 255 + k).  m and v are rounded to leading bits at random, up with the
probability that leaves their expectation as it was, by 16 random bits for each value that are a function of
(seed, t, index); a v below the lowest code is kept at the lowest."""
import math
import random

import torch

own = False

BLOCK = 256                    # elements that share the leading bits of an 8-bit moment; tensors start at multiples
GOLDEN = 0x9E3779B97F4A7C15
MASK = (1 << 64) - 1
BETAS, LR, EPS, DECAY = (0.9, 0.999), 1e-3, 1e-8, 0.01
DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


# ---- cases ---------------------------------------------------------------------------------------------------------
def _gn(name, n, c, groups, h, w, dtype='float32', act='relu', residual=True, train=False, wide_affine=True):
    return dict(name=name, op='group_norm', n=n, c=c, groups=groups, h=h, w=w, dtype=dtype, act=act, residual=residual,
                train=train, wide_affine=wide_affine)


def _adamw(name, kind, blocks, channels, shared, bits, dtype='float32', count=0, tensors_seed=0, most=0):
    return dict(name=name, op='adamw', kind=kind, blocks=blocks, channels=channels, shared=shared, bits=bits, dtype=dtype,
                count=count, tensors_seed=tensors_seed, most=most)


def listed():
    return [
        # one position in front of the default 256-channel tower, as a single game's search evaluates it: latency
        _gn('gn_one_position', 1, 256, 32, 6, 7),
        # the leaves of 8192 concurrent games in a 128-channel tower: inference at the self-play batch
        _gn('gn_leaves_8192', 8192, 128, 16, 6, 7),
        # feature planes larger than a board, few of them: a sample's group is far more than one workgroup holds
        _gn('gn_planes_64x64_bf16', 3, 320, 32, 64, 64, dtype='bfloat16', act='silu', residual=False),
        # the second norm of a residual block in a training step at the shipped batch of 128, default width
        _gn('gn_step_128', 128, 256, 32, 6, 7, train=True),
        # the same in 16 bits at a batch that fills the card
        _gn('gn_step_4096_bf16', 4096, 128, 16, 6, 7, dtype='bfloat16', train=True),
        # a large odd board, odd batch, 12 channels to a group
        _gn('gn_step_19x19_fp16', 61, 192, 16, 19, 19, dtype='float16', act='silu', residual=False, train=True, wide_affine=False),
        # the policy head's two planes, one group, no residual
        _gn('gn_step_head', 4096, 2, 1, 6, 7, residual=False, train=True),
        # the shipped 6 x 32 Connect Four network: 22 tensors, the smallest step
        _adamw('adamw_6x32', 'net', 6, 32, True, 32),
        # the default 39 x 256 network (one block's tensors, applied 39 times), moments in 8 bits
        _adamw('adamw_39x256_8bit', 'net', 39, 256, True, 8),
        # a 39 x 256 tower whose blocks have tensors of their own: bandwidth, 32 and 8 bits
        _adamw('adamw_tower_32bit', 'net', 39, 256, False, 32),
        _adamw('adamw_tower_8bit', 'net', 39, 256, False, 8),
        # bfloat16 parameters with a master copy, many tensors of ragged sizes
        _adamw('adamw_ragged_bf16', 'ragged', 0, 0, False, 32, dtype='bfloat16', count=157, tensors_seed=3, most=300000),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    if rng.random() < 0.6:
        train = rng.random() < 0.6
        h, w = (rng.choice([(3, 3), (6, 7), (1, 1), (19, 19)]) if rng.random() < 0.4 else
                (_log_int(rng, 1, 64), _log_int(rng, 1, 64)))
        if rng.random() < 0.7:
            groups, per = rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([1, 2, 4, 8, 16])
        else:
            groups, per = rng.randint(1, 24), rng.randint(1, 24)
        c = groups * per
        most = (20 if train else 40) * 1000 * 1000 // (c * h * w)
        case = _gn('', _log_int(rng, 1, max(1, min(8192, most))), c, groups, h, w, dtype=rng.choice(list(DTYPES)),
                   act=rng.choice(['relu', 'relu', 'silu', 'none']), residual=rng.random() < 0.5, train=train,
                   wide_affine=rng.random() < 0.5)
    elif rng.random() < 0.5:
        shared = rng.random() < 0.4
        case = _adamw('', 'net', rng.randint(1, 39), rng.choice([4, 8, 16, 32, 48, 64, 100, 128, 192, 256]), shared,
                      rng.choice([8, 32]), dtype=rng.choice(['float32', 'float32', 'bfloat16']))
    else:
        case = _adamw('', 'ragged', 0, 0, False, rng.choice([8, 32]), dtype=rng.choice(['float32', 'bfloat16']),
                      count=_log_int(rng, 1, 300), tensors_seed=rng.randrange(1 << 20), most=_log_int(rng, 1, 1000000))
        if case['count'] * case['most'] > 80 * 1000 * 1000:
            case['most'] = 80 * 1000 * 1000 // case['count']
    del case['name']
    return case


def _shapes(case):
    """Tensor shapes in the order of the two parameter groups: those with weight decay (two or more dimensions), then
    those without."""
    if case['kind'] == 'ragged':
        rng = random.Random(case['tensors_seed'])
        sizes = [_log_int(rng, 1, case['most']) for _ in range(case['count'])]
        shapes = [(s, 1) if rng.random() < 0.7 else (s,) for s in sizes]
    else:
        c, cells = case['channels'], 42
        shapes = [(c, 2, 3, 3), (c,), (c,)]
        shapes += [(c, c, 3, 3), (c,), (c,), (c, c, 3, 3), (c,), (c,)] * (1 if case['shared'] else case['blocks'])
        shapes += [(2, c, 1, 1), (2,), (2,), (2,), (cells, 2 * cells), (cells,)]
        shapes += [(1, c, 1, 1), (1,), (1,), (256, cells), (256,), (1, 256), (1,)]
    return [s for s in shapes if len(s) > 1], [s for s in shapes if len(s) == 1]


def _blocks_of(shapes):
    return [-(-math.prod(s) // BLOCK) for s in shapes]


# ---- inputs --------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device='cuda', generator=gen)  # noqa: E731
    if case['op'] == 'group_norm':
        n, c, h, w = case['n'], case['c'], case['h'], case['w']
        dtype = DTYPES[case['dtype']]
        affine = torch.float32 if case['wide_affine'] else dtype
        # what a convolution leaves: channels of different spread and offset
        spread, offset = torch.exp(0.5 * normal(c)), 0.5 * normal(c)
        plane = lambda: normal(n, h, w, c).to(dtype).permute(0, 3, 1, 2)  # noqa: E731
        s = {'case': case, 'x': (normal(n, h, w, c) * spread + offset).to(dtype).permute(0, 3, 1, 2),
             'weight': (1 + 0.2 * normal(c)).to(affine), 'bias': (0.2 * normal(c)).to(affine),
             'residual': plane().relu() if case['residual'] else None}
        if case['train']:
            s['dy'] = plane()
            for k in ('x', 'weight', 'bias', 'residual'):
                if s[k] is not None:
                    s[k].requires_grad_()
        return s
    decayed, plain = _shapes(case)
    shapes = decayed + plain
    blocks = _blocks_of(shapes)
    total = sum(blocks)
    size = torch.tensor([math.prod(s) for s in shapes], device='cuda')
    owner = torch.repeat_interleave(torch.arange(len(shapes), device='cuda'), torch.tensor(blocks, device='cuda'))
    first = torch.cumsum(torch.tensor([0] + blocks[:-1], device='cuda'), 0)
    place = (torch.arange(total, device='cuda') - first[owner])[:, None] * BLOCK + torch.arange(BLOCK, device='cuda')
    inside = (place < size[owner][:, None]).float()
    # gradients of a trained network: each tensor of its own size, some entries zero (inputs that never fire)
    level = torch.exp(1.5 * normal(len(shapes)) - 7)[owner][:, None]
    fires = (torch.rand(total, BLOCK, device='cuda', generator=gen) > 0.1).float() * inside
    dtype = DTYPES[case['dtype']]
    p = (0.05 * normal(total, BLOCK) * inside).to(dtype)
    g = (level * normal(total, BLOCK) * fires).to(dtype)
    m = 0.3 * level * normal(total, BLOCK) * inside
    v = (level * torch.exp(0.7 * normal(total, BLOCK))) ** 2 * fires
    bound = sum(_blocks_of(decayed))
    s = {'case': case, 'p': p.float(), 'g': g, 't': 1 + seed % 997, 'seed': seed % (1 << 31),
         'decay': torch.where(torch.arange(total, device='cuda') < bound, DECAY, 0.0)[:, None]}
    if dtype != torch.float32:
        s['p16'] = p
    if case['bits'] == 8:
        half = torch.full((total, BLOCK), 1 << 15, device='cuda', dtype=torch.int32)
        s['m8'], s['m_top'] = _encode_m(m, half)
        s['v8'], s['v_top'] = _encode_v(v, half)
        m, v = _decode_m(s['m8'], s['m_top']), _decode_v(s['v8'], s['v_top'])
    if own:
        s['optimizer'] = _own_optimizer(s, decayed, plain, p, m, v)
    if case['bits'] == 32:
        s['m'], s['v'] = m, v
    return s


def _cut(flat, shapes):
    """The tensors of `shapes` out of the padded buffer."""
    flat, out, at = flat.reshape(-1), [], 0
    for s, b in zip(shapes, _blocks_of(shapes)):
        out.append(flat[at:at + math.prod(s)].reshape(s))
        at += b * BLOCK
    return out


def _own_optimizer(s, decayed, plain, p, m, v):
    from alphazero_amd.optim import FlatAdamW
    case, shapes = s['case'], decayed + plain
    params = [torch.nn.Parameter(t.clone()) for t in _cut(p, shapes)]
    groups = [dict(params=q, weight_decay=d) for q, d in ((params[:len(decayed)], DECAY), (params[len(decayed):], 0.0)) if q]
    opt = FlatAdamW(groups, lr=LR, betas=BETAS, eps=EPS, state_bits=case['bits'], seed=s['seed'])
    state = opt.state_dict()
    for i, (a, b, master) in enumerate(zip(_cut(m, shapes), _cut(v, shapes), _cut(s['p'], shapes))):
        state['state'][i] = dict(step=s['t'], exp_avg=a, exp_avg_sq=b)
        if 'p16' in s:
            state['state'][i]['master'] = master
    opt.load_state_dict(state)
    for q, grad in zip(params, _cut(s['g'], shapes)):
        q.grad.copy_(grad)
    return opt


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(s):
    if s['case']['op'] == 'adamw':
        return _own_adamw(s) if own else _plain_adamw(s)
    if own:
        return _own_norm(s)
    return _plain_norm_step(s) if s['case']['train'] else {'y': _plain_norm(s)}


def _own_norm(s):
    from alphazero_amd.norm import group_norm_act
    case = s['case']
    y = group_norm_act(s['x'], case['groups'], s['weight'], s['bias'], act=case['act'], residual=s['residual'])
    if not case['train']:
        return {'y': y}
    leaves = [k for k in ('x', 'weight', 'bias', 'residual') if s[k] is not None]
    grads = torch.autograd.grad(y, [s[k] for k in leaves], s['dy'])
    return {'y': y.detach(), **{'d' + k: g for k, g in zip(leaves, grads)}}


def _own_adamw(s):
    opt = s['optimizer']
    opt.step()
    m, v = opt.state_values()
    out = {'p': opt.flat_p, 'm': m, 'v': v}
    if 'p16' in s:
        out['p16'] = opt.flat_p16
    return out


def _grouped(t, groups):
    """[N, C, H, W] -> [N, H * W, G, C / G], in memory's order for channels last."""
    n, c, h, w = t.shape
    return t.permute(0, 2, 3, 1).reshape(n, h * w, groups, c // groups)


def _planes(t, like):
    n, c, h, w = like.shape
    return t.reshape(n, h, w, c).permute(0, 3, 1, 2)


def _activation(z, act):
    if act == 'relu':
        return torch.where(z > 0, z, torch.zeros_like(z))
    return z / (1 + torch.exp(-z)) if act == 'silu' else z


def _normalised(s, dtype):
    """(xhat, rstd, z) in `dtype`."""
    groups = s['case']['groups']
    x = _grouped(s['x'].detach(), groups).to(dtype)
    weight, bias = (s[k].detach().to(dtype).view(groups, -1) for k in ('weight', 'bias'))
    mean = x.mean((1, 3), keepdim=True)
    centred = x - mean
    rstd = 1 / torch.sqrt((centred * centred).mean((1, 3), keepdim=True) + 1e-5)
    xhat = centred * rstd
    z = xhat * weight + bias
    if s['residual'] is not None:
        z = z + _grouped(s['residual'].detach(), groups).to(dtype)
    return xhat, rstd, z


def _plain_norm(s):
    z = _normalised(s, torch.float32)[2]
    return _planes(_activation(z, s['case']['act']), s['x']).to(s['x'].dtype)


def _plain_norm_step(s):
    case, x = s['case'], s['x'].detach()
    # relu cuts the gradient where z passes zero, and a value next to that border falls on the right side of it only
    # in 64 bits; the other activations have no border
    xhat, rstd, z = _normalised(s, torch.float64 if case['act'] == 'relu' else torch.float32)
    open_ = z > 0
    xhat, rstd, z = xhat.float(), rstd.float(), z.float()
    y = _activation(z, case['act'])
    dz = _grouped(s['dy'], case['groups']).float()
    if case['act'] == 'relu':
        dz = torch.where(open_, dz, torch.zeros_like(dz))
    elif case['act'] == 'silu':
        sig = 1 / (1 + torch.exp(-z))
        dz = dz * (sig * (1 + z * (1 - sig)))
    weight = s['weight'].detach().float().view(case['groups'], -1)
    dbias, dweight = dz.sum((0, 1)), (dz * xhat).sum((0, 1))
    a = dz * weight
    dx = rstd * (a - a.mean((1, 3), keepdim=True) - xhat * (a * xhat).mean((1, 3), keepdim=True))
    out = {'y': _planes(y, x).to(x.dtype), 'dx': _planes(dx, x).to(x.dtype),
           'dweight': dweight.reshape(-1).to(s['weight'].dtype), 'dbias': dbias.reshape(-1).to(s['bias'].dtype)}
    if s['residual'] is not None:
        out['dresidual'] = _planes(dz, x).to(x.dtype)
    return out


def _plain_adamw(s):
    b1, b2 = BETAS
    s['t'] += 1
    t, g = s['t'], s['g'].float()
    if s['case']['bits'] == 8:
        m, v = _decode_m(s['m8'], s['m_top']), _decode_v(s['v8'], s['v_top'])
    else:
        m, v = s['m'], s['v']
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    p = s['p'] * (1 - LR * s['decay']) - (LR / (1 - b1 ** t)) * m / (torch.sqrt(v) / math.sqrt(1 - b2 ** t) + EPS)
    s['p'] = p
    if s['case']['bits'] == 8:
        rm, rv = _random_bits(s['seed'], t, m.numel(), m.device)
        s['m8'], s['m_top'] = _encode_m(m, rm)
        s['v8'], s['v_top'] = _encode_v(v, rv)
        m, v = _decode_m(s['m8'], s['m_top']), _decode_v(s['v8'], s['v_top'])
    else:
        s['m'], s['v'] = m, v
    out = {'p': p.reshape(-1), 'm': m.reshape(-1), 'v': v.reshape(-1)}
    if 'p16' in s:
        out['p16'] = p.to(s['p16'].dtype).reshape(-1)
    return out


# ---- moments in 8 bits ---------------------------------------------------------------------------------------------
def _mix(z):
    """splitmix64's output function, of a whole number or (two's complement) of int64 values."""
    if isinstance(z, int):
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & MASK
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & MASK
        return z ^ (z >> 31)
    after = lambda v, k: (v >> k) & ((1 << (64 - k)) - 1)  # noqa: E731
    z = (z ^ after(z, 30)) * _signed(0xBF58476D1CE4E5B9)
    z = (z ^ after(z, 27)) * _signed(0x94D049BB133111EB)
    return z ^ after(z, 31)


def _signed(u):
    return u - (1 << 64) if u >> 63 else u


def _random_bits(seed, t, count, device):
    """16 bits for each of `count` elements, for m and for v: two 64-bit numbers for every four elements."""
    key = _mix((seed + GOLDEN * t) & MASK)
    counter = torch.arange(count // 2, device=device, dtype=torch.int64)
    z = _mix(counter * _signed(GOLDEN) + _signed(key)).reshape(-1, 2, 1)
    bits = (z >> torch.tensor([0, 16, 32, 48], device=device)) & 0xFFFF
    return tuple(bits[:, k].reshape(-1, BLOCK).to(torch.int32) for k in (0, 1))


def _leading(x, random_bits, codes):
    """(rounded leading bits of |x|, the block's top, the lowest leading bits that have a code, |x| as bits)"""
    a = x.abs().contiguous().view(torch.int32)
    top = (a.amax(1, keepdim=True) + 0xFFFFF) >> 20
    return (a + (random_bits << 4)) >> 20, top, (top - (codes - 1)).clamp(min=1), a


def _encode_m(x, random_bits):
    q, top, lowest, a = _leading(x, random_bits, 127)
    up = x.abs() * 131072 > (2 * random_bits + 1).float() * (lowest << 20).view(torch.float32)
    k = torch.where(q >= lowest, q - (top - 127), torch.where(up, lowest - (top - 127), 0))
    return (k | torch.where((x < 0) & (k > 0), 128, 0)).to(torch.uint8), top.to(torch.int16)


def _encode_v(x, random_bits):
    q, top, lowest, a = _leading(x, random_bits, 255)
    k = torch.where(a > 0, torch.maximum(q, lowest) - (top - 255), 0)
    return k.to(torch.uint8), top.to(torch.int16)


def _decode_m(code, top):
    k = (code & 127).to(torch.int32)
    x = torch.where(k > 0, (k + top.to(torch.int32) - 127) << 20, 0).view(torch.float32)
    return torch.where(code > 127, -x, x)


def _decode_v(code, top):
    k = code.to(torch.int32)
    return torch.where(k > 0, (k + top.to(torch.int32) - 255) << 20, 0).view(torch.float32)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    if case['op'] == 'group_norm':
        size = DTYPES[case['dtype']].itemsize
        values = case['n'] * case['c'] * case['h'] * case['w']
        affine = 2 * case['c'] * (4 if case['wide_affine'] else size)
        planes = 2 + case['residual']
        if not case['train']:
            return {'bytes': values * size * planes + affine, 'flops': 8 * values}
        return {'bytes': values * size * (planes + 2 + case['residual']) + 2 * affine, 'flops': 24 * values}
    values = sum(math.prod(s) for part in _shapes(case) for s in part)
    param = 8 + 4 if case['dtype'] == 'float32' else 8 + 2 + 2
    # in 8 bits the moments' codes are read and written, and the values that they stand for are handed out
    moments = 16 if case['bits'] == 32 else 4 + 8
    return {'bytes': values * (param + moments), 'flops': 16 * values}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'adamw':
        p, g = s['p'].double(), s['g'].double()
        wide = case['bits'] == 32
        m = (s['m'] if wide else _decode_m(s['m8'], s['m_top'])).double()
        v = (s['v'] if wide else _decode_v(s['v8'], s['v_top'])).double()
        t = s['t'] + 1
        m = m + (1 - BETAS[0]) * (g - m)
        v = v + (1 - BETAS[1]) * (g.square() - v)
        ahead = m / (1 - BETAS[0] ** t)
        spread = (v / (1 - BETAS[1] ** t)).sqrt()
        p = p - LR * (s['decay'].double() * p + ahead / (spread + EPS))
        out = {'p': p.flatten(), 'm': m.flatten() if wide else None, 'v': v.flatten() if wide else None}
        if 'p16' in s:
            out['p16'] = out['p']
        return out
    n, c, h, w = s['x'].shape
    leaf = lambda k: s[k].detach().double().requires_grad_(case['train'])  # noqa: E731
    x, weight, bias = leaf('x'), leaf('weight'), leaf('bias')
    r = leaf('residual') if s['residual'] is not None else None
    rows = x.reshape(n, case['groups'], -1)
    var, mean = torch.var_mean(rows, 2, correction=0, keepdim=True)
    z = ((rows - mean) / (var + 1e-5).sqrt()).reshape(n, c, h, w) * weight[:, None, None] + bias[:, None, None]
    if r is not None:
        z = z + r
    y = z.clamp(min=0) if case['act'] == 'relu' else z * torch.sigmoid(z) if case['act'] == 'silu' else z
    if not case['train']:
        return {'y': y}
    names = ['x', 'weight', 'bias'] + (['residual'] if r is not None else [])
    grads = torch.autograd.grad(y, [x, weight, bias] + ([r] if r is not None else []), s['dy'].double())
    return {'y': y.detach(), **{'d' + k: d for k, d in zip(names, grads)}}
