"""The operators of latent attention on the host: what the C entry points refuse before they touch a device, what the Python functions refuse, and the
reference implementation that the GPU tests compare with, against torch's attention and its gradients."""
import ctypes

import pytest
import torch
import torch.nn.functional as F

import attention_reference as R
from conftest import load_package


@pytest.fixture(scope="module")
def pkg():
    return load_package()


def _struct(first_ints, size=640):
    """A zeroed argument struct whose leading 32-bit fields are given."""
    buf = (ctypes.c_int32 * (size // 4))()
    for i, v in enumerate(first_ints):
        buf[i] = v
    return buf


ENTRIES = {   # dtype and sizes that are refused as a shape
    "el_rotary": [[1, 2, 3, 4, 7]],                                                        # batch, length, heads, dim
    "el_latent_attention": [[1, 2, 3, 4, 5, 200, 57, 8], [1, 2, 3, 4, 5, 64, 0, 257]],     # batch, length, keys, heads, key_dim, rot_dim, value_dim
    "el_latent_attention_backward": [[1, 2, 3, 4, 5, 200, 57, 8], [1, 2, 3, 4, 5, 64, 0, 257]],
    "el_latent_cache_write": [[1, 2, 3, 24, 0, 4, 16, 1], [1, 2, 3, 528, 0, 4, 16, 1], [1, 2, 3, 64, 65, 4, 16, 1], [1, 2, 3, 64, 0, 4, 0, 1]],   # .., rank, rot_dim, pages, page_size
    "el_latent_cache_read": [[1, 2, 3, 24, 0, 4, 16, 1], [1, 2, 3, 528, 0, 4, 16, 1], [1, 2, 3, 0, 0, 4, 16, 1]],
    "el_latent_attention_step": [[1, 2, 4, 64, 0, 64, 24, 4, 16], [1, 2, 4, 257, 0, 64, 64, 4, 16], [1, 2, 4, 64, 65, 64, 64, 4, 16], [1, 2, 4, 64, 0, 64, 64, 4, 0]],
}


@pytest.mark.parametrize("name", sorted(ENTRIES))
def test_entry_points_refuse_on_the_host(pkg, name):
    lib, fn = pkg._lib, getattr(pkg._lib.lib(), name)
    assert fn(None, None) == lib.EL_ERR_NULL_PTR
    assert fn(_struct([9]), None) == lib.EL_ERR_INVALID_ARG                    # dtype
    assert fn(_struct([lib.EL_BF16, -1]), None) == lib.EL_ERR_INVALID_ARG      # a negative size
    for sizes in ENTRIES[name]:
        assert fn(_struct(sizes), None) == lib.EL_ERR_UNSUPPORTED_SHAPE, sizes


def test_sizes_that_the_kernels_cannot_count_are_refused(pkg):
    lib, h = pkg._lib, pkg._lib.lib()
    assert h.el_latent_attention(_struct([1, 1 << 20, 1 << 20, 1, 1 << 10, 64, 0, 64]), None) == lib.EL_ERR_TOO_LARGE
    assert h.el_latent_attention(_struct([1, 1, 0x7FFFFFFF, 1, 1, 64, 0, 64]), None) == lib.EL_ERR_TOO_LARGE
    assert h.el_latent_attention_step(_struct([1, 65536, 4, 64, 0, 64, 64, 4, 16, 1]), None) == lib.EL_ERR_TOO_LARGE
    assert h.el_latent_cache_read(_struct([1, 1 << 20, 1 << 20, 64, 0, 4, 16, 1]), None) == lib.EL_ERR_TOO_LARGE


def test_workspace_sizes(pkg):
    h = pkg._lib.lib()
    bad = _struct([9])
    for name in ("el_latent_attention_lse_bytes", "el_latent_attention_backward_workspace_bytes", "el_latent_attention_step_workspace_bytes"):
        assert getattr(h, name)(bad) == 0
    # a float32 for every query of every head, rows padded to 128
    assert h.el_latent_attention_lse_bytes(_struct([1, 2, 129, 300, 5, 64, 0, 64])) == 2 * 5 * 256 * 4


@pytest.mark.parametrize("call,message", [
    (lambda o, t: o.latent_attention(t[:, None], t), "q must be a CUDA tensor"),
    (lambda o, t: o.latent_attention(t[:, None].requires_grad_(True), t), "q must be a CUDA tensor"),
    (lambda o, t: o.rotary(t, t), "x must be a CUDA tensor"),
    (lambda o, t: o.rotary(t, t.clone().requires_grad_(True)), "no gradient of its table"),
    (lambda o, t: o.latent_cache_write(o.LatentCache(t, t, t), t, t), "latent must be a CUDA tensor"),
    (lambda o, t: o.latent_cache_read(o.LatentCache(t, t, t), t, 3), "latents must be a CUDA tensor"),
    (lambda o, t: o.latent_attention_step(t, t, 1.0, o.LatentCache(t, t, t), t, t, 8), "q must be a CUDA tensor"),
    (lambda o, t: o.latent_attention_step(t.requires_grad_(True), t, 1.0, o.LatentCache(t, t, t), t, t, 8), "no gradient"),
    (lambda o, t: o.rotary_table(4, 5), "even"),
])
def test_python_functions_refuse(pkg, call, message):
    with pytest.raises(RuntimeError, match=message):
        call(pkg.attention_ops, torch.zeros(2, 3, 8))


def test_reference_attention_is_torchs():
    g = torch.Generator().manual_seed(0)
    B, T, H, D, P, V = 2, 9, 3, 8, 4, 6
    q, kv, qr, kr = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((B, T, H, D), (B, T, H * (D + V)), (B, T, H, P), (B, T, P)))
    dout = torch.randn(B, T, H, V, generator=g, dtype=torch.float64)
    k, v = kv[..., :H * D].unflatten(-1, (H, D)), kv[..., H * D:].unflatten(-1, (H, V))
    out = F.scaled_dot_product_attention(torch.cat([q, qr], -1).transpose(1, 2), torch.cat([k, kr[:, :, None].expand(-1, -1, H, -1)], -1).transpose(1, 2), v.transpose(1, 2), is_causal=True)
    grads = torch.autograd.grad(out, (q, kv, qr, kr), dout.transpose(1, 2))
    value, bound = R.attention(q.detach(), kv.detach(), qr.detach(), kr.detach(), True, None, None, None, torch.float32, dout)
    assert torch.allclose(value["out"], out.detach().transpose(1, 2), rtol=0, atol=1e-13)
    for name, want in zip(("dq", "dkv", "dq_rot", "dk_rot"), grads):
        assert torch.allclose(value[name], want, rtol=0, atol=1e-13), name
        assert (bound[name] >= 0).all()


def test_reference_rotation_keeps_lengths_and_differences():
    g = torch.Generator().manual_seed(1)
    pkg = load_package()
    table = pkg.attention_ops.rotary_table(50, 8)
    x, y = torch.randn(8, generator=g, dtype=torch.float64), torch.randn(8, generator=g, dtype=torch.float64)
    for neighbours in (False, True):
        turned = [R.rotate(x, table, torch.tensor(p), neighbours) @ R.rotate(y, table, torch.tensor(p + 5), neighbours) for p in (0, 17, 44)]
        assert max(turned) - min(turned) < 1e-6            # the table is float32


def test_reference_step_is_the_expanded_form():
    g = torch.Generator().manual_seed(2)
    B, H, D, V, rank, page, n = 1, 2, 8, 4, 16, 3, 7
    latents, absmax = torch.randint(-128, 128, (4, page, rank), generator=g).to(torch.int8), torch.rand(4, page, generator=g)
    blocks, W, q = torch.tensor([[2, 0, 3]]), torch.randint(-1, 2, (H * (D + V), rank), generator=g), torch.randn(B, H, D, generator=g)
    out, _ = R.step(q, W, 0.3, latents, absmax, None, blocks, torch.tensor([n]), V, None, None, None, torch.float32)
    c, _, here, _ = R.cached(latents, absmax, None, blocks[0], n)
    assert here.all()
    kv = (c @ W.double().T * 0.3)[None]
    value, _ = R.attention(q[:, None], kv, None, None, True, None, None, None, torch.float32)
    assert torch.allclose(out, value["out"][:, 0], rtol=0, atol=1e-13)
