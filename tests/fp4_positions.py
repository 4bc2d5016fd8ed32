"""A position encoding of its own for the tests of four-bit pages, and a model of two layers with it."""
from glassbox_amd import ops
from glassbox_amd.parts.base import PositionEncoding, TensorSpec


class Learned(PositionEncoding):
    """A table row per position is added to every query and key head; key heads that are not stored are left as they are."""

    def __init__(self, head_dim, positions):
        self.head_dim, self.positions = head_dim, positions

    def tensor_specs(self):
        return {"position_table": TensorSpec((self.positions, self.head_dim), kind="f32")}

    def load(self, tensors):
        self.table = tensors["position_table"]

    def add(self, ctx, qkv, heads, head_dim):
        moved = qkv.view(qkv.shape[0], -1, head_dim)[:, :heads]
        moved.copy_((moved.float() + self.table[ctx.positions.long()][:, None]).to(qkv.dtype))

    def apply_and_store(self, ctx, qkv, n_heads, n_kv_heads, head_dim, slots, k_pages, v_pages):
        self.add(ctx, qkv, n_heads + (n_kv_heads if slots is not None else 0), head_dim)
        if slots is not None:
            ops.rope_store(qkv, None, None, slots, k_pages, v_pages, n_heads, n_kv_heads, head_dim, rotate=False, portions=ctx.portions())


class LearnedInPlace(Learned):
    def apply(self, ctx, qkv, n_heads, n_kv_heads, head_dim):
        self.add(ctx, qkv, n_heads + n_kv_heads, head_dim)


def model_of(positions, d=96, H=6, G=2, D=64, vocab=90, eps=1e-5):
    """A layer for each of the encodings."""
    import helpers
    from glassbox_amd.config import config_from_dict
    from glassbox_amd.parts.attention import PagedAttention
    from glassbox_amd.parts.block import PreNormBlock
    from glassbox_amd.parts.embedding import Embedding, LMHead
    from glassbox_amd.parts.mlp import SwiGLU
    from glassbox_amd.parts.model import DecoderModel, LayerCall
    from glassbox_amd.parts.norm import RMSNorm
    embedding = Embedding(vocab, d)
    cfg = config_from_dict(dict(helpers.TINY_B, hidden_size=d, intermediate_size=160, num_hidden_layers=len(positions), num_attention_heads=H,
                                num_key_value_heads=G, head_dim=D, vocab_size=vocab, rms_norm_eps=eps, tie_word_embeddings=True))
    blocks = [PreNormBlock(RMSNorm(d, eps), PagedAttention(d, H, G, D, position), RMSNorm(d, eps), SwiGLU(d, 160)) for position in positions]
    return DecoderModel(cfg, embedding, blocks, [LayerCall(i, cache=i) for i in range(len(positions))], RMSNorm(d, eps),
                        LMHead(vocab, d, tied_to=embedding))
