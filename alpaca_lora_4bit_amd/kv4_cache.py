"""The key/value cache of many requests: a pool of pages of 4-bit keys and values per layer, shared by all sequences.

The reference keeps one dense fp16 cache per `generate` call (transformers' own, inference.py:33-44); a 4-bit weight file leaves the cache as the
largest tensor of a server, so here it is held in 4 bits as well: a sign, two bits of exponent and one of mantissa per value and one fp16 scale
per `group` dimensions of a token and head, 4 + 16 / group bits a value.  `quant_hip.kv4_append`, `kv4_read` and `kv4_attention` work on it; the
byte order is written out in include/q4_gptq.h.
"""
import torch

from . import quant_hip


def new_layer(pages, heads, head_dim, page=64, group=32, device="cuda"):
    """(k_codes, v_codes, k_scales, v_scales) of one layer: `pages` pages of `page` tokens (a multiple of 16, up to 1024) of `heads` key heads of
    `head_dim` (64 or 128) dimensions with a scale per `group` (32, 64 or 128) of them; zeros."""
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, not {head_dim}")
    if group not in (32, 64, 128) or group > head_dim:
        raise ValueError(f"group must be 32, 64 or 128 and at most head_dim, not {group}")
    if page < 16 or page > 1024 or page % 16:
        raise ValueError(f"page must be a multiple of 16 up to 1024, not {page}")
    if pages < 1 or heads < 1:
        raise ValueError("pages and heads must be positive")
    codes = dict(dtype=torch.int32, device=device)
    scales = dict(dtype=torch.float16, device=device)
    return (torch.zeros((pages, heads, page, head_dim // 8), **codes), torch.zeros((pages, heads, page // 4, head_dim // 8, 4), **codes),
            torch.zeros((pages, heads, head_dim // group, page), **scales), torch.zeros((pages, heads, head_dim // group, page), **scales))


def rope_table(rotary_emb, positions, device="cuda"):
    """fp32 [positions, rotated / 2, 2]: the cosines and sines that a model's rotary embedding module gives for positions 0 .. positions - 1, as
    `kv4_append` takes them (pairs (i, i + rotated / 2) have the same angle, so the first half of the module's columns holds them all)."""
    kind = getattr(rotary_emb, "rope_type", "default")
    if kind in ("dynamic", "longrope"):
        raise ValueError(f"rotary embedding of type {kind!r}: its angles depend on the sequence's length, a table by position cannot hold them")
    at = torch.arange(positions, device=device)[None]
    with torch.no_grad(), torch.autocast(torch.device(device).type, enabled=False):
        cos, sin = rotary_emb(torch.empty(1, dtype=torch.float32, device=device), at)
    half = cos.shape[-1] // 2
    return torch.stack((cos[0, :, :half].float(), sin[0, :, :half].float()), dim=-1).contiguous()


class PagedKv4Cache:
    """The layers' pools and which pages are free.  A request takes its pages with `open` and gives them back with `close`; the tokens themselves
    are written by `quant_hip.kv4_append` at the places that a table of `table` names."""

    def __init__(self, layers, heads, head_dim, pages, page=64, group=32, device="cuda"):
        self.page = page
        self.layers = [new_layer(pages, heads, head_dim, page, group, device) for _ in range(layers)]
        self.device = self.layers[0][0].device if self.layers else torch.device(device)
        self._free = list(range(pages - 1, -1, -1))

    @property
    def free_pages(self):
        return len(self._free)

    def pages_for(self, tokens):
        return -(-tokens // self.page)

    def open(self, tokens):
        """Pages for a request of up to `tokens` tokens, as a list of page numbers that is its handle."""
        need = self.pages_for(tokens)
        if need > len(self._free):
            raise RuntimeError(f"{tokens} tokens need {need} pages, {len(self._free)} are free")
        return [self._free.pop() for _ in range(need)]

    def close(self, handle):
        """Takes the pages of a handle back (and empties it: a second close gives nothing back twice)."""
        self._free.extend(reversed(handle))
        del handle[:]

    def table(self, handles):
        """int32 [requests, pages of the longest]: the page tables of these requests; -1 where a request has no page."""
        width = max([len(h) for h in handles] + [1])
        return torch.tensor([list(h) + [-1] * (width - len(h)) for h in handles], dtype=torch.int32).to(self.device)

    def read(self, layer, handle, tokens):
        """(k, v) fp16 [tokens, heads, head_dim]: the first `tokens` tokens of a request in one layer, for a caller that goes on with dense keys
        and values."""
        if not 0 <= tokens <= len(handle) * self.page:
            raise ValueError(f"{tokens} tokens are not in {len(handle)} pages of {self.page}")
        lengths = torch.tensor([tokens], dtype=torch.int32).to(self.device)
        return quant_hip.kv4_read(self.layers[layer], self.table([handle]), lengths, tokens)
