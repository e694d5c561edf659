"""Speculative decoding with draft trees: the tree, the verification of its
tokens and the acceptance of a path."""

from engine.decode.draft import DraftTree, Verified, accept_draft, draft_tree, verify_draft, verify_greedy

__all__ = ["DraftTree", "Verified", "accept_draft", "draft_tree", "verify_draft", "verify_greedy"]
