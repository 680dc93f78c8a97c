"""Answering from a trained model: recurrent state per conversation, prompts, single tokens, sampling."""
from .generate import Generator, load_weights
from .state import DecodeState, get_serving, serving

__all__ = ["DecodeState", "Generator", "get_serving", "load_weights", "serving"]
