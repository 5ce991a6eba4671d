"""8-bit key/value cache of a decoder on the GPU, and the attention that reads it.

The cache is blocks of BLOCK_SIZE tokens.  For each (block, head) the keys share one float32 scale and the values another;
value = code * scale with codes in [-127, 127].  Half the memory and half the traffic of a float16 cache.

A batch is described by three int32 tensors on the device, which no call waits for:
    offsets [B + 1]      rows offsets[b] ... offsets[b + 1] - 1 of k, v, q and the result are the newest tokens of sequence b
    seq_lens [B]         its length with them: its last row has position seq_lens[b] - 1
    block_table [B, W]   token t of sequence b lies in block block_table[b, t // BLOCK_SIZE] of the cache
A sequence with more rows than tokens is padded in front: those rows are not stored and attend to nothing (zeros).  Rows from
offsets[B] on are neither read nor written.  A block number outside the cache is a block that is not there: nothing is stored in
it and attention passes over its tokens.  Two sequences may read the same block; a batch may append to it at one place of the
table only.
"""
import ctypes

from popxl_addons import _gq_hip

__all__ = ["BLOCK_SIZE", "KVCacheGQ", "kv_cache_append", "kv_cache_attention", "kv_cache_gather"]

BLOCK_SIZE = 64


class KVCacheGQ:
    """The cache of one layer: k_codes uint8 [n_blocks, kv_heads, BLOCK_SIZE, head_dim], v_codes uint8 [n_blocks, kv_heads,
    head_dim, BLOCK_SIZE] (transposed: the product with the probabilities contracts over tokens), both holding code + 128, and
    k_scale, v_scale float32 [n_blocks, kv_heads].  head_dim is a multiple of 16, at most 256.  Any blocks can be handed to any
    sequence; what a block held before does not matter to a sequence that starts in it."""

    def __init__(self, n_blocks, kv_heads, head_dim, device="cuda"):
        import torch

        if head_dim % 16 != 0 or not 16 <= head_dim <= 256:
            raise ValueError(f"KVCacheGQ: head_dim={head_dim} must be a multiple of 16 up to 256")
        if n_blocks < 0 or kv_heads < 1:
            raise ValueError(f"KVCacheGQ: n_blocks={n_blocks}, kv_heads={kv_heads}")
        self._adopt(torch.full((n_blocks, kv_heads, BLOCK_SIZE, head_dim), 128, dtype=torch.uint8, device=device),
                    torch.full((n_blocks, kv_heads, head_dim, BLOCK_SIZE), 128, dtype=torch.uint8, device=device),
                    torch.zeros((n_blocks, kv_heads), dtype=torch.float32, device=device),
                    torch.zeros((n_blocks, kv_heads), dtype=torch.float32, device=device))

    @classmethod
    def from_tensors(cls, k_codes, v_codes, k_scale, v_scale):
        """A cache on tensors that exist (not copied).  Scales are not negative; tokens under a scale of 0 are zeros, whatever
        their codes."""
        import torch

        self = cls.__new__(cls)
        if k_codes.dim() != 4 or k_codes.shape[2] != BLOCK_SIZE:
            raise ValueError(f"KVCacheGQ: k_codes must be [n_blocks, kv_heads, {BLOCK_SIZE}, head_dim], got {tuple(k_codes.shape)}")
        n_blocks, kv_heads, _, head_dim = k_codes.shape
        if head_dim % 16 != 0 or not 16 <= head_dim <= 256:
            raise ValueError(f"KVCacheGQ: head_dim={head_dim} must be a multiple of 16 up to 256")
        if tuple(v_codes.shape) != (n_blocks, kv_heads, head_dim, BLOCK_SIZE):
            raise ValueError(f"KVCacheGQ: v_codes must be {(n_blocks, kv_heads, head_dim, BLOCK_SIZE)}, got {tuple(v_codes.shape)}")
        for scale in (k_scale, v_scale):
            if tuple(scale.shape) != (n_blocks, kv_heads):
                raise ValueError(f"KVCacheGQ: scales must be {(n_blocks, kv_heads)}, got {tuple(scale.shape)}")
            if scale.dtype != torch.float32:
                raise TypeError("KVCacheGQ: scales must be float32")
        if k_codes.dtype != torch.uint8 or v_codes.dtype != torch.uint8:
            raise TypeError("KVCacheGQ: codes must be uint8")
        for t in (k_codes, v_codes, k_scale, v_scale):
            if not t.is_contiguous() or t.device != k_codes.device:
                raise ValueError("KVCacheGQ: the cache's tensors must be contiguous and on one device")
        self._adopt(k_codes, v_codes, k_scale, v_scale)
        return self

    def _adopt(self, k_codes, v_codes, k_scale, v_scale):
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale
        self.n_blocks, self.kv_heads, _, self.head_dim = k_codes.shape
        self.device, self.index = k_codes.device, k_codes.get_device()
        self._c = _gq_hip.KvCache(*(t.data_ptr() for t in (k_codes, v_codes, k_scale, v_scale)), self.n_blocks, self.kv_heads,
                                  self.head_dim)
        self._attention_workspace = _gq_hip.load().gq_kv_attention_workspace_bytes(self.head_dim)


def _batch(cache, offsets, seq_lens, block_table, tokens):
    """The batch for the C entry points, and the tensors to keep until the call has been made."""
    import torch

    index = cache.index
    if index < 0:
        raise RuntimeError("the key/value cache runs on the GPU only: make it on a HIP device")
    for name, t in (("offsets", offsets), ("seq_lens", seq_lens), ("block_table", block_table)):
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, got {t.dtype}")
        if t.get_device() != index:
            raise ValueError(f"{name} must be on the cache's device")
    sequences = seq_lens.shape[0] if seq_lens.dim() == 1 else -1
    if sequences < 0 or offsets.dim() != 1 or offsets.shape[0] != sequences + 1:
        raise ValueError(f"offsets must have one entry more than seq_lens, got {tuple(offsets.shape)} and {tuple(seq_lens.shape)}")
    if block_table.dim() != 2 or block_table.shape[0] != sequences:
        raise ValueError(f"block_table must be [{sequences}, blocks], got {tuple(block_table.shape)}")
    offsets, seq_lens, block_table = keep = offsets.contiguous(), seq_lens.contiguous(), block_table.contiguous()
    return _gq_hip.KvBatch(offsets.data_ptr(), seq_lens.data_ptr(), block_table.data_ptr(), sequences, block_table.shape[1], tokens), keep


def _rows(name, t, cache, heads):
    """t [tokens, heads, head_dim] float16 with rows that the kernels can load (a copy where they cannot), and its strides."""
    import torch

    if t.dim() != 3 or t.shape[2] != cache.head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [tokens, {heads if heads is not None else 'heads'}, {cache.head_dim}], got {tuple(t.shape)}")
    if t.dtype != torch.float16:
        raise TypeError(f"{name} must be float16, got {t.dtype}")
    if t.get_device() != cache.index:
        raise ValueError(f"{name} must be on the cache's device")
    token_stride, head_stride, stride = t.stride()
    if stride != 1 or token_stride % 8 or head_stride % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        token_stride, head_stride, _ = t.stride()
    return t, token_stride, head_stride


def kv_cache_append(cache, k, v, offsets, seq_lens, block_table, rotary=None):
    """
    Store the newest tokens of every sequence.

    Args:
        cache (KVCacheGQ): changed in place
        k, v (torch.Tensor): float16 [tokens, kv_heads, head_dim], the last axis contiguous: slices of a fused projection's result
            are read where they lie
        offsets, seq_lens, block_table: the batch (see the module)
        rotary (RotaryPosEmbed): turn the keys by their positions on the way, with the bits that `rotary_pos_embed` would give

    A block that starts with these tokens gets the scale amax / 127.  In a block that has tokens the scale grows, where it must,
    by a power of two, and the codes there are scaled down by it: every value stays within one scale of what was stored.
    """
    batch, keep = _batch(cache, offsets, seq_lens, block_table, k.shape[0])
    if k.shape != v.shape:
        raise ValueError(f"k and v must have the same shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    k, k_token_stride, k_head_stride = _rows("k", k, cache, cache.kv_heads)
    v, v_token_stride, v_head_stride = _rows("v", v, cache, cache.kv_heads)
    if rotary is not None:
        if rotary.index != cache.index:
            raise ValueError("rotary must be on the cache's device")
        if rotary.rotary_dim > cache.head_dim:
            raise ValueError(f"rotary_dim={rotary.rotary_dim} exceeds the head dimension {cache.head_dim}")
    _gq_hip.launch(cache.index, "gq_kv_append_f16", ctypes.byref(cache._c), ctypes.byref(batch), k.data_ptr(), k_token_stride,
                   k_head_stride, v.data_ptr(), v_token_stride, v_head_stride, None if rotary is None else rotary.argument)


def kv_cache_gather(cache, offsets, seq_lens, block_table, tokens, out=None):
    """
    Read tokens back: (k, v) float16 [tokens, kv_heads, head_dim] for the rows that the batch describes (a whole sequence is read
    with offsets that give it seq_lens[b] rows).  Rows of no token or of a block that is not there are not written: they
    keep what the contiguous tensors `out` = (k, v) hold, and hold nothing in particular without `out`.
    """
    import torch

    batch, keep = _batch(cache, offsets, seq_lens, block_table, tokens)
    shape = (tokens, cache.kv_heads, cache.head_dim)
    if out is None:
        out = (torch.empty(shape, dtype=torch.float16, device=cache.device), torch.empty(shape, dtype=torch.float16, device=cache.device))
    k, v = out
    for t in out:
        if t.shape != shape or not t.is_contiguous() or t.dtype != torch.float16 or t.get_device() != cache.index:
            raise ValueError(f"out must be two contiguous float16 tensors of shape {shape} on the cache's device")
    _gq_hip.launch(cache.index, "gq_kv_gather_f16", ctypes.byref(cache._c), ctypes.byref(batch), k.data_ptr(), v.data_ptr())
    return out


def kv_cache_attention(q, cache, offsets, seq_lens, block_table, scale=None, out=None):
    """
    Causal attention of the newest tokens of every sequence over its cache (append them first).

    Args:
        q (torch.Tensor): float16 [tokens, q_heads, head_dim], the last axis contiguous; query head i reads kv head
            i // (q_heads / kv_heads)
        offsets, seq_lens, block_table: the batch (see the module)
        scale (float): of the scores, head_dim ** -0.5 if None
        out (torch.Tensor): float16, the shape of q, apart from it (q itself is refused); a new tensor if None, whose rows from
            offsets[B] on hold nothing in particular

    Returns:
        torch.Tensor: `out`.  Decode steps, prompts in chunks and mixtures of both are one call; results do not depend on timing.  (One
        kernel takes the whole batch, chosen by its rows a sequence on average: decode steps with long histories beside a long chunk
        take about half the time as two calls.)
    """
    import torch

    batch, keep = _batch(cache, offsets, seq_lens, block_table, q.shape[0])
    q, q_token_stride, q_head_stride = _rows("q", q, cache, None)
    shape = q.shape
    if shape[1] % cache.kv_heads != 0:
        raise ValueError(f"q has {shape[1]} heads, not a multiple of the cache's {cache.kv_heads}")
    if out is None:
        out = q.new_empty(shape)
    elif out.shape != shape or out.stride(2) != 1 or out.get_device() != cache.index:
        raise ValueError("out must have the shape and device of q and a contiguous last axis")
    elif out.dtype != torch.float16:
        raise TypeError("out must be float16")
    if shape[1] == 0:
        return out
    token_stride, head_stride, _ = out.stride()
    workspace = torch.empty(cache._attention_workspace, dtype=torch.uint8, device=cache.device)
    _gq_hip.launch(cache.index, "gq_kv_attention_f16", ctypes.byref(cache._c), ctypes.byref(batch), q.data_ptr(), q_token_stride,
                   q_head_stride, out.data_ptr(), token_stride, head_stride, shape[1], cache.head_dim ** -0.5 if scale is None else scale,
                   workspace.data_ptr(), cache._attention_workspace)
    return out
