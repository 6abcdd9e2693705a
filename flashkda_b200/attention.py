"""Linear attention with a decay for each head, and latent attention: the layers that stand beside KDA layers in a model.

Same manner as ``fwd``: outputs are allocated by the caller and written in place, work is enqueued on the current CUDA stream
of ``q.device`` without synchronising, there is no gradient and no CPU path, and a call that is refused raises
``RuntimeError`` before anything is enqueued.  Tensors may be views (a slice of a fused projection, a layout with heads in front of
tokens): the last dimension is contiguous, the others are any positive multiples of 8 elements apart, on 16-byte addresses.  Outputs
overlap no inputs (a linear call's two states may be one buffer).
"""
import torch

from . import _lib


def _host():
    """The native host side; there is no other implementation, so a missing build is an error."""
    _lib.lib()   # the CUDA library, with its own error when it has not been built
    try:
        from . import _host as host
    except ImportError as e:
        raise RuntimeError("flashkda_b200/_host.so is missing or does not load: build it with "
                           f"`python -m flashkda_b200.build` ({e})") from e
    return host


def _bind(name):
    def first(*args):
        globals()[f"_{name}"] = call = getattr(_host(), name)
        return call(*args)
    return first


_linear_attention_fwd = _bind("linear_attention_fwd")
_latent_attention_fwd = _bind("latent_attention_fwd")
_latent_attention_decode = _bind("latent_attention_decode")


def linear_attention_fwd(q, k, v, g, scale, out, initial_state=None, final_state=None, cu_seqlens=None, *, workspace: torch.Tensor = None):
    """Linear attention with a decay for each head; writes ``out`` (and ``final_state``) in place and returns ``None``::

        S_t = exp(g_t) S_{t-1} + v_t k_t^T        o_t = scale S_t q_t

    q, k: bf16 ``[B, T, Hk, 128]``; v, out: bf16 ``[B, T, H, 128]``, where ``Hk`` divides ``H`` and value head ``h`` reads
    key head ``h // (H // Hk)``; g: fp32 ``[B, T, H]``, natural logarithms of the decays, or ``[H]``, one constant for each head
    (any strides; meant for values up to 0, below -100 counts as -100, so minus infinity starts a sequence afresh); states: bf16
    or fp32 ``[N, H, 128, 128]`` (``[V, K]`` layout, as ``fwd``'s), which may be the same buffer; cu_seqlens: int64 ``[N + 1]``
    (then ``B`` must be 1).  Rows of ``out`` that no sequence has are left as they were.

    Sequences of more than one token go through 64-token chunks on the tensor cores; single tokens (``T == 1``, or the sequences of one
    token in a packed batch of mostly such) through one read-modify-write of the states.  In between the state is fp32, whatever its type
    in memory; what a chunk adds to it holds 24 bits, or 16 behind a bf16 ``initial_state``, and the sums are cut off, not rounded (1e-6 of a
    state that remembers 256 tokens, 3e-5 for 8 192).  Outputs do not depend on whether a
    ``final_state`` is asked for, nor on its type.  An element of v that is not finite makes its dimension of out NaN from the start of its
    chunk on, so in up to 63 tokens in front of it; of q, k and g nothing reaches an earlier token.  ``workspace``: optional caller-owned uint8 scratch for calls that need some
    (``linear_attention_workspace_size``).
    """
    _linear_attention_fwd(q, k, v, g, scale, out, initial_state, final_state, cu_seqlens, workspace)


def latent_attention_fwd(q, k, k_rope, v, scale, out, lse=None, cu_seqlens=None, cu_seqlens_k=None, *, causal: bool = True):
    """Latent attention of prompts, expanded form; writes ``out`` (and ``lse``) in place and returns ``None``::

        o_i = sum_j softmax_j(scale (q_i[:128] . k_j + q_i[128:] . k_rope_j)) v_j

    q: bf16 ``[B, T, H, 192]`` (128 unrotated, then 64 rotated dimensions); k, v: bf16 ``[B, Tk, H, 128]``, every head's own;
    k_rope: bf16 ``[B, Tk, 64]``, the token's, shared by the heads; out: bf16 ``[B, T, H, 128]``; lse: fp32 ``[B, T, H]``, the
    logarithm of the softmax's sum, with which results over parts of the keys can be joined.  ``causal``: query ``i`` of ``T`` sees
    the keys ``j <= i + Tk - T`` (the last query sees all: keys in front of the queries are a cached prefix); a row that sees nothing
    gets 0 and ``lse`` minus infinity.  cu_seqlens, cu_seqlens_k: int64 ``[N + 1]`` of packed queries and keys (then ``B`` must
    be 1); ``cu_seqlens`` serves both if it is given alone.  Rows that no sequence has are left as they were.  An element of v that is
    not finite makes its dimension of out NaN also in rows that do not see it, up to 255 in front of those that do; of k and k_rope nothing
    reaches such rows.  ``scale`` must be positive.
    """
    _latent_attention_fwd(q, k, k_rope, v, scale, out, lse, cu_seqlens, cu_seqlens_k, causal)


def latent_attention_decode(q, cache, block_table, cache_lens, scale, out, lse=None, *, workspace: torch.Tensor = None):
    """Latent attention of the newest tokens over a paged cache, absorbed form; writes ``out`` (and ``lse``) in place and returns
    ``None``::

        o_r = sum_j softmax_j(scale q_r . c_j) c_j[:512]

    q: bf16 ``[B, Tq, H, 576]``, the ``Tq`` newest tokens of every sequence, multiplied by the expansion of the keys (512) and
    beside it their rotated part (64); cache: bf16 ``[pages, page_size, 576]``, a token's latent vector and its rotated key,
    ``page_size`` a multiple of 16; block_table: int32 ``[B, max_pages]``, a sequence's pages in order; cache_lens: int32 ``[B]``,
    tokens in the cache, the new ones among them; out: bf16 ``[B, Tq, H, 512]``; lse: fp32 ``[B, Tq, H]``.  New token ``i`` sees the
    first ``len - Tq + 1 + i`` tokens; one that sees none gets 0 and ``lse`` minus infinity.  In q and out the new tokens lie ``H``
    heads apart.  What a page holds behind a sequence's last token is not used; entries of ``block_table`` that are no page number
    read page 0.  A cached number among a token's first 512 that is not finite makes its dimension of out NaN for all ``Tq`` tokens of its
    sequence, those that do not see it as well.  At most 36 864 sequences; ``scale`` must be positive.  ``workspace``: optional caller-owned uint8 scratch
    (``latent_decode_workspace_size``).
    """
    _latent_attention_decode(q, cache, block_table, cache_lens, scale, out, lse, workspace)


def linear_attention_workspace_size(B: int, T: int, H: int, N: int = None, packed: bool = False) -> int:
    """Scratch bytes of a ``linear_attention_fwd`` call on v of shape ``[B, T, H, 128]`` (``packed``: with ``N`` sequences)."""
    p = _lib.LinearParams(B=int(B), T=int(T), H=int(H), Hk=int(H), N=int(B if N is None else N), cu_seqlens=256 if packed else None)
    return int(_lib.lib().fkda_linear_workspace_bytes(p))


def latent_decode_workspace_size(B: int, Tq: int, H: int) -> int:
    """Scratch bytes of a ``latent_attention_decode`` call on q of shape ``[B, Tq, H, 576]``, whatever the cache's size."""
    return int(_lib.lib().fkda_latent_decode_workspace_bytes(_lib.LatentDecodeParams(B=int(B), Tq=int(Tq), H=int(H))))


def operator_status(device=None) -> int:
    """Synchronises the current stream of ``device`` and returns 0, or the status code of a kernel of these operators, on whatever stream
    and of whatever thread, that gave up on one of its bounded internal waits there since this thread last asked (the first time: since the
    library was loaded; see ``device_status`` for ``fwd``)."""
    with torch.cuda.device(device):
        return int(_lib.lib().fkda_operator_status(torch.cuda.current_stream().cuda_stream))
