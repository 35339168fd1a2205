"""Inputs of the tests of the paged cache."""
import torch

DEV = 'cuda'


def cache(pages, page_size, heads, dim, dtype, seed=0, layout='slots'):
    """k_cache, v_cache [pages, page_size, heads, dim]; layout 'heads': a page's heads lie in front of its slots; 'one': keys and values in one tensor, between 16-byte
    boundaries where the element size says so."""
    gen = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(pages, page_size, heads, dim, generator=gen).to(dtype).to(DEV) for _ in range(2))
    if layout == 'heads':
        return tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    if layout == 'one':
        both = torch.zeros(pages, 2, page_size, heads, dim, dtype=dtype, device=DEV)
        both[:, 0], both[:, 1] = k, v
        return both[:, 0], both[:, 1]
    if layout == 'odd':
        wide = torch.zeros(pages, page_size, heads, dim + 3, dtype=dtype, device=DEV)
        wide2 = wide.clone()
        wide[..., 1:dim + 1], wide2[..., 2:dim + 2] = k, v
        return wide[..., 1:dim + 1], wide2[..., 2:dim + 2]
    return k, v


def table(lengths, page_size, pages, seed=0, extra=1):
    """[N, pages of the longest + extra] int32: pages in any order, -1 behind a sequence's last."""
    need = [-(-n // page_size) for n in lengths]
    assert sum(need) <= pages, (need, pages)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    t = torch.full((len(lengths), max(need) + extra), -1, dtype=torch.int32)
    for n, count in enumerate(need):
        t[n, :count] = torch.tensor(order[:count], dtype=torch.int32)
        order = order[count:]
    return t


def pages_for(lengths, page_size):
    return sum(-(-n // page_size) for n in lengths) + 2
