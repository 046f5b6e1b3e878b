"""Lists of gradients at their ends: what the host calls write, and what the device calls refuse before anything is launched (no GPU needed)."""
import torch

P = 0x10000        # an address that is never read: these calls launch nothing


def fill(cf, counts, to, size):
    n = len(counts)
    c, p, t = torch.tensor(counts, dtype=torch.int64), torch.full((n,), P, dtype=torch.int64), torch.ones(n, dtype=torch.int32)
    return cf.raw_cf_grad_list_fill(p.data_ptr(), None, c.data_ptr(), t.data_ptr(), n, to, size)


def test_bytes_to_clear_need_a_list(cf):
    """Tensors without elements need no entry, but the bytes that the size names are cleared: there has to be memory for them."""
    for size in (1, 32, 64, 4096):
        assert fill(cf, [0, 0], None, size) == -1
        assert cf.raw_cf_grad_list_fill(None, None, None, None, 0, None, size) == -1
    assert fill(cf, [0, 0], None, 0) == 0 and cf.raw_cf_grad_list_fill(None, None, None, None, 0, None, 0) == 0
    image = torch.full((96,), 0xa5, dtype=torch.uint8)
    assert fill(cf, [0, 0], image.data_ptr(), 64) == 0
    assert bool((image[:64] == 0).all()) and bool((image[64:] == 0xa5).all())


def test_lists_that_32_bits_do_not_walk(cf):
    """A workgroup's walk steps over the entries in 32 bits, up to 2048 + 4096 beyond the last one: a list of that many less than 2^32 would never end."""
    for entries in (2 ** 31, 2 ** 32 - 4096, 2 ** 32 - 1, 2 ** 32):
        assert cf.raw_cf_grad_norm(P, entries * 32, P, P, 1 << 20, None) == -1
        assert cf.raw_cf_grad_clip(P, entries * 32, 1.0, P, None, None) == -1
        assert cf.raw_cf_grad_norm_clip(P, entries * 32, 1.0, P, None, P, 1 << 20, None) == -1
