"""Plain CPU forms of the rotation and of the 4-bit page format for the tests of
rope_kv_append, rope_kv_append_int4, kv_gather_int4 and paged_decode_attention_int4."""
import torch

PLANE = 64


def angles(positions, rot, base=10000.0):
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def rotate(x, cos, sin, interleaved):
    """x [N, H, D] turned by cos/sin [N, rot / 2], in x's own precision, each product and sum
    rounded on its own."""
    rot = 2 * cos.shape[-1]
    c, s = cos.to(x.dtype)[:, None], sin.to(x.dtype)[:, None]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        y[..., : rot // 2], y[..., rot // 2 : rot] = a * c - b * s, b * c + a * s
    return y


def quantise(x):
    """fp32 [..., D] -> (codes uint8 [..., D], params fp16 [..., D / 64, 2])."""
    g = x.unflatten(-1, (-1, PLANE))
    least, most = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((most - least) / 15.0).clamp(max=65504.0).half()
    zero = least.clamp(-65504.0, 65504.0).half()
    q = ((g - zero.float()) / scale.float()).round().clamp(0, 15)
    codes = torch.where(scale > 0, q, torch.zeros_like(q)).nan_to_num(0.0).to(torch.uint8)
    return codes.flatten(-2), torch.cat((scale, zero), -1)


def values(codes, params):
    """The float64 values that codes [..., D] and params [..., D / 64, 2] stand for."""
    g = codes.unflatten(-1, (-1, PLANE)).double()
    return (g * params[..., :1].double() + params[..., 1:].double()).flatten(-2)


def pack(k_codes, k_params, v_codes, v_params):
    """codes [blocks, bs, H, D] and params [blocks, bs, H, P, 2] -> the uint8 pool."""
    parts = []
    for codes, params in ((k_codes, k_params), (v_codes, v_params)):
        both = codes[..., 0::2] + 16 * codes[..., 1::2]
        both = both.unflatten(-1, (-1, PLANE // 2))                          # [blocks, bs, H, P, 32]
        parts.append(both.permute(0, 2, 3, 1, 4).reshape(codes.shape[0], codes.shape[2], -1))
        parts.append(params.permute(0, 2, 3, 1, 4).contiguous().view(torch.uint8).reshape(
            codes.shape[0], codes.shape[2], -1))
    return torch.cat(parts, -1).contiguous()


def unpack(pool, D, bs):
    """The pool -> (k_codes, k_params, v_codes, v_params), the inverse of pack()."""
    P, out = D // PLANE, []
    nc, np_ = P * bs * 32, P * bs * 4
    for o in (0, nc + np_):
        c = pool[..., o : o + nc].reshape(*pool.shape[:2], P, bs, 32).permute(0, 3, 1, 2, 4)
        out.append(torch.stack((c & 15, c >> 4), -1).flatten(-2).flatten(-2))
        s = pool[..., o + nc : o + nc + np_].contiguous().view(torch.float16)
        out.append(s.reshape(*pool.shape[:2], P, bs, 2).permute(0, 3, 1, 2, 4))
    return out


def random_pool(gen, blocks, bs, H, D, spread=1.0):
    """A pool of quantised normal values: (pool, k float64, v float64 [blocks, bs, H, D])."""
    made = []
    for _ in range(2):
        made += list(quantise(torch.randn(blocks, bs, H, D, generator=gen) * spread))
    kc, kp, vc, vp = made
    return pack(kc, kp, vc, vp), values(kc, kp), values(vc, vp)


def tables(gen, lens, bs, spare=3):
    """int32 [B, max blocks] over a shuffled pool, and the pool's number of blocks."""
    most = max(1, max(-(-n // bs) for n in lens))
    blocks = len(lens) * most + spare
    return torch.randperm(blocks, generator=gen)[: len(lens) * most].view(len(lens), most).to(torch.int32), blocks


def cu(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32).cumsum(0, dtype=torch.int32)
