"""Sinkhorn and local attention operators backed by libdfsink.so."""
