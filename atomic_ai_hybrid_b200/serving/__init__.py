"""Answering from a trained model: recurrent state per conversation, prompts, single tokens, sampling."""
from .generate import Generator, compute_weights, load_weights
from .state import DecodeState, get_serving, serving

__all__ = ["DecodeState", "Generator", "compute_weights", "get_serving", "load_weights", "serving"]
